"""Attention over parts of a latent context in 64 bits, straight from the formulas, with the error bounds of the kernels
against it. Rounding units and their counts are those of tests/latent_reference.py."""

from __future__ import annotations

import math

import torch

from tests.latent_reference import E, F64, U


def seen_by_window(n, L, window, sinks, device="cuda"):
    """[n, L]: query i, at position L - n + i, sees its last `window` keys and the first `sinks`."""
    p = (L - n + torch.arange(n, device=device))[:, None]
    j = torch.arange(L, device=device)[None, :]
    return (j <= p) & ((j > p - window) | (j < sinks))


def lines(parents, cap=1 << 30):
    """Of each node the nodes on its line to the root, itself first; nodes from `cap` on have none."""
    out = []
    for i in range(len(parents)):
        line, at = [], i if i < cap else -1
        while at >= 0:
            line.append(at)
            at = parents[at] if 0 <= parents[at] < at else -1
        out.append(line)
    return out


def seen_by_tree(parents, L, window=None, sinks=0, words=16, device="cuda"):
    """[n, L]: the last n of L tokens are the nodes."""
    n = len(parents)
    base, cap = L - n, 64 * words
    keep = torch.zeros((n, L), dtype=torch.bool)
    for i, line in enumerate(lines(parents, cap)):
        depth = max(len(line) - 1, 0)
        for j in range(max(base, 0)):
            keep[i, j] = window is None or j > base + depth - window or j < sinks
        for a in line:
            if base + a >= 0:
                keep[i, base + a] = True
    return keep.to(device)


def attend(q, k, v, scale, keep):
    """One sequence's rows: q [r, D], k [L, D], v [L, V] in 64 bits, keep [r, L]. Returns out, lse and the bounds of both,
    as latent_reference.attend derives them."""
    r, L = keep.shape
    zero = torch.zeros((), dtype=F64, device=q.device)
    if L == 0:
        z = torch.zeros((r, v.shape[1]), dtype=F64, device=q.device)
        return z, torch.full((r,), -math.inf, dtype=F64, device=q.device), z, torch.zeros(r, dtype=F64, device=q.device)
    s = torch.where(keep, q @ k.T.contiguous() * scale, zero - math.inf)
    ds = (torch.where(keep, q.abs() @ k.abs().T.contiguous() * scale, zero) * ((q.shape[1] + 8) * E)).amax(-1, keepdim=True)
    lse = torch.logsumexp(s, -1)
    p = torch.where(keep, (s - torch.where(lse == -math.inf, zero, lse)[:, None]).exp(), zero)
    out, mag = p @ v, p @ v.abs()
    return out, lse, U * out.abs() + (U + 4 * ds + (L + 64) * E) * mag + 1e-30, \
        2 * ds[:, 0] + (L + 64) * E + 4 * E * torch.nan_to_num(lse, neginf=0.0).abs()


def absorbed(q_latent, q_rope, rows, starts, scale, keeps):
    """rows[b]: the cached rows of sequence b as values; keeps[b] [n, L]."""
    T, H, R = q_latent.shape
    out = torch.zeros((T, H, R), dtype=F64, device=q_latent.device)
    lse = torch.full((T, H), -math.inf, dtype=F64, device=q_latent.device)
    tol, ltol = torch.zeros_like(out), torch.zeros((T, H), dtype=F64, device=q_latent.device)
    q = q_latent.to(F64) if q_rope is None else torch.cat([q_latent.to(F64), q_rope.to(F64)], -1)
    for b, keep in enumerate(keeps):
        lo, hi = starts[b], starts[b + 1]
        k = rows[b][:keep.shape[1]].to(F64)
        o, s, t, u = attend(q[lo:hi].reshape(-1, q.shape[-1]), k, k[:, :R], scale, keep.repeat_interleave(H, 0))
        out[lo:hi], lse[lo:hi], tol[lo:hi], ltol[lo:hi] = (x.reshape(hi - lo, H, *x.shape[1:]) for x in (o, s, t, u))
    return out, lse, tol, ltol


def expanded(q, kv, k_rope, q_starts, kv_starts, scale, keeps):
    T, H, D = q.shape
    P = 0 if k_rope is None else k_rope.shape[1]
    N = D - P
    V = kv.shape[2] - N
    out = torch.zeros((T, H, V), dtype=F64, device=q.device)
    lse = torch.full((T, H), -math.inf, dtype=F64, device=q.device)
    tol, ltol = torch.zeros_like(out), torch.zeros((T, H), dtype=F64, device=q.device)
    for b, keep in enumerate(keeps):
        lo, hi, k0, k1 = q_starts[b], q_starts[b + 1], kv_starts[b], kv_starts[b + 1]
        for h in range(H):
            k = kv[k0:k1, h, :N].to(F64)
            if P:
                k = torch.cat([k, k_rope[k0:k1].to(F64)], 1)
            o, s, t, u = attend(q[lo:hi, h].to(F64), k, kv[k0:k1, h, N:].to(F64), scale, keep)
            out[lo:hi, h], lse[lo:hi, h], tol[lo:hi, h], ltol[lo:hi, h] = o, s, t, u
    return out, lse, tol, ltol


def weights(q_latent, q_rope, rows, kv_lens, starts, lse, scale, positions, previous):
    """[B, positions] and its bound: a weight errs by its score's error, that of lse in binary32 as log2 and of the
    exponent itself (8 roundings of the larger of the two), relative to itself; the sum over r rows by r E of it; the
    addition to what was there by one rounding."""
    B, (T, H) = len(kv_lens), lse.shape
    out = torch.zeros((B, positions), dtype=F64, device=lse.device) if previous is None else previous.to(F64).clone()
    tol = E * out.abs() + 1e-37
    q = q_latent.to(F64) if q_rope is None else torch.cat([q_latent.to(F64), q_rope.to(F64)], -1)
    for b, L in enumerate(kv_lens):
        lo, hi = starts[b], starts[b + 1]
        n, m = hi - lo, min(L, positions)
        if n <= 0 or L == 0:
            continue
        k = rows[b][:L].to(F64)
        x = q[lo:hi].reshape(n * H, -1)
        s = x @ k.T.contiguous() * scale
        mag = x.abs() @ k.abs().T.contiguous() * scale * ((x.shape[1] + 8) * E)
        mine = lse[lo:hi].reshape(-1, 1).to(F64)
        keep = seen_by_window(n, L, L + n + 1, 0, lse.device).repeat_interleave(H, 0) & (mine != -math.inf)
        p = torch.where(keep, (s - torch.where(keep, mine, 0 * mine)).exp(), 0 * s)
        a = p.sum(0)
        dp = torch.where(keep, p * (2 * mag + 16 * E * (s.abs() + torch.where(keep, mine, 0 * mine).abs() + 1)), 0 * s).sum(0)
        out[b, :m] += a[:m]
        tol[b, :m] += (dp + (n * H + 64) * E * a)[:m] + E * out[b, :m].abs()
    return out, tol


def heaviest(weights_, length, keep, sinks, recent):
    """Positions that stay, by sorting in Python."""
    length = max(0, min(length, len(weights_)))
    if length <= keep:
        return list(range(length))
    last = length - recent
    middle = sorted(range(sinks, last), key=lambda j: (-math.inf if math.isnan(weights_[j]) else 0, -weights_[j]
                                                       if not math.isnan(weights_[j]) else 0, j))
    return sorted([*range(sinks), *middle[:keep - sinks - recent], *range(last, length)])
