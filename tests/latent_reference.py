"""Latent attention in 64 bits, straight from the formulas, and the error bounds of the kernels against it.

Rounding to bf16 is off by at most U = 2^-8 relative, to e4m3 by 2^-4 (half a subnormal step, 2^-10, below 2^-6); a
binary32 operation by E = 2^-24. Bounds count the roundings the operators document: sums of n terms n E of the sum of
magnitudes, one rounding of the softmax weights to bf16, one of the output.
"""

from __future__ import annotations

import math

import torch

U = 2.0 ** -8
E = 2.0 ** -24
F64 = torch.float64


def rope_table(P, count, device="cpu", base=10000.0):
    a = torch.arange(count, dtype=F64, device=device)[:, None] * base ** (
        -torch.arange(0, max(P, 1), 2, dtype=F64, device=device)[None, : P // 2] / max(P, 1))
    return torch.cat([a.cos(), a.sin()], 1).float().contiguous()


def rotate(x, rows, interleaved, inverse):
    """x [T, ..., D] in 64 bits, table rows [T, P]; also the magnitude |a| + |b| behind each value."""
    P = rows.shape[1]
    if P == 0:
        return x, x.abs()
    rows = rows.to(F64).reshape(rows.shape[0], *([1] * (x.dim() - 2)), P)
    cos, sin = rows[..., : P // 2], rows[..., P // 2:] * (-1 if inverse else 1)
    tail = x[..., x.shape[-1] - P:]
    a, b = (tail[..., 0::2], tail[..., 1::2]) if interleaved else (tail[..., : P // 2], tail[..., P // 2:])
    ra, rb, mag = a * cos - b * sin, b * cos + a * sin, a.abs() + b.abs()
    join = (lambda u, v: torch.stack([u, v], -1).flatten(-2)) if interleaved else (lambda u, v: torch.cat([u, v], -1))
    keep = x[..., : x.shape[-1] - P]
    return torch.cat([keep, join(ra, rb)], -1), torch.cat([keep.abs(), join(mag, mag)], -1)


def norm(x, weight, eps):
    y = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    return y if weight is None else y * weight.to(F64)


def attend(q, k, v, scale, limits):
    """One head's rows: q [n, D], k [L, D], v [L, V] in 64 bits, row i sees keys 0 .. limits[i]. Returns out, lse and
    the bounds of both: the scores' error is at most D E of their products' magnitudes (each weight errs by as much,
    relative to itself), the weights and the result are rounded to bf16."""
    n, L = q.shape[0], k.shape[0]
    keep = torch.arange(L, device=q.device)[None, :] < limits[:, None]
    inf = torch.tensor(math.inf, dtype=F64, device=q.device)
    s = torch.where(keep, q @ k.T.contiguous() * scale, -inf)
    ds = (torch.where(keep, q.abs() @ k.abs().T.contiguous() * scale, 0 * inf.new_zeros(())) * ((q.shape[1] + 8) * E)
          ).amax(-1, keepdim=True) if L else torch.zeros((n, 1), dtype=F64, device=q.device)
    if L == 0:
        z = torch.zeros((n, v.shape[1]), dtype=F64, device=q.device)
        return z, torch.full((n,), -math.inf, dtype=F64, device=q.device), z, torch.zeros(n, dtype=F64, device=q.device)
    lse = torch.logsumexp(s, -1)
    p = torch.where(keep, (s - torch.where(lse == -math.inf, torch.zeros_like(lse), lse)[:, None]).exp(), 0 * s.new_zeros(()))
    out, mag = p @ v, p @ v.abs()
    return out, lse, U * out.abs() + (U + 4 * ds + (L + 64) * E) * mag + 1e-30, \
        2 * ds[:, 0] + (L + 64) * E + 4 * E * torch.nan_to_num(lse, neginf=0.0).abs()


def limits(n, L, causal=True, device="cpu"):
    i = torch.arange(n, device=device)
    return (L - n + i + 1).clamp(0, L) if causal else torch.full((n,), L, device=device)


def absorbed(q_latent, q_rope, rows, kv_lens, starts, scale):
    """rows[b]: the cached rows of sequence b [L, R + P] as values."""
    T, H, R = q_latent.shape
    out = torch.zeros((T, H, R), dtype=F64, device=q_latent.device)
    lse = torch.full((T, H), -math.inf, dtype=F64, device=q_latent.device)
    tol, ltol = torch.zeros_like(out), torch.zeros((T, H), dtype=F64, device=q_latent.device)
    q = q_latent.to(F64) if q_rope is None else torch.cat([q_latent.to(F64), q_rope.to(F64)], -1)
    for b, L in enumerate(kv_lens):
        lo, hi = starts[b], starts[b + 1]
        k = rows[b][:L].to(F64)
        lim = limits(hi - lo, L, device=q.device).repeat_interleave(H)
        o, s, t, u = attend(q[lo:hi].reshape(-1, q.shape[-1]), k, k[:, :R], scale, lim)
        out[lo:hi], lse[lo:hi], tol[lo:hi], ltol[lo:hi] = (x.reshape(hi - lo, H, *x.shape[1:]) for x in (o, s, t, u))
    return out, lse, tol, ltol


def expanded(q, kv, k_rope, q_starts, kv_starts, scale, causal):
    T, H, D = q.shape
    P = 0 if k_rope is None else k_rope.shape[1]
    N = D - P
    V = kv.shape[2] - N
    out = torch.zeros((T, H, V), dtype=F64, device=q.device)
    lse = torch.full((T, H), -math.inf, dtype=F64, device=q.device)
    tol, ltol = torch.zeros_like(out), torch.zeros((T, H), dtype=F64, device=q.device)
    for b in range(len(q_starts) - 1):
        lo, hi, k0, k1 = q_starts[b], q_starts[b + 1], kv_starts[b], kv_starts[b + 1]
        lim = limits(hi - lo, k1 - k0, causal, device=q.device)
        for h in range(H):
            k = kv[k0:k1, h, :N].to(F64)
            if P:
                k = torch.cat([k, k_rope[k0:k1].to(F64)], 1)
            o, s, t, u = attend(q[lo:hi, h].to(F64), k, kv[k0:k1, h, N:].to(F64), scale, lim)
            out[lo:hi, h], lse[lo:hi, h], tol[lo:hi, h], ltol[lo:hi, h] = o, s, t, u
    return out, lse, tol, ltol


def assert_within(got, want, tol, what=""):
    got = got.to(F64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine), f"{what}: finite values differ"
    assert torch.equal(got[~fine].nan_to_num(nan=7.0), want[~fine].nan_to_num(nan=7.0)), f"{what}: other values differ"
    over = ((got - want).abs() - tol)[fine]
    if over.numel():
        worst = int(over.argmax())
        assert float(over.max()) <= 0, (f"{what}: {int((over > 0).sum())} of {over.numel()} values past their bound, worst "
                                        f"{float(got[fine][worst])} for {float(want[fine][worst])}, bound "
                                        f"{float(tol[fine][worst])}")
