"""The measured work of ``fused_cpp_amd.latent_attention``: the steps of a latent-attention layer between its
W8A8 projections, each through its public entry point.

A case is a dict of plain values with an ``op``:

* ``norm_rope``: per-head RMS norm and position rotation of ``[T, H, D]`` rows.
* ``append``: normalise, rotate and write ``T`` latent rows into a paged cache (``dtype`` bf16 or e4m3).
* ``project``: the per-head products ``[T, H, K] x [H, N, K]`` around the absorbed form.
* ``absorbed``: attention of ``n`` query tokens a sequence over a paged latent cache, lengths ``low..high``.
* ``expanded``: causal attention over per-head keys and values, ``B`` sequences of up to ``T`` new tokens with
  ``past`` earlier keys each.

``own`` picks the framework's kernels; without it ``run`` computes the operators from elementary operations in
32 bits.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
_E4M3_MAX = 448.0

# The layer that the repository's W8A8 projections belong to (wq_b N = 24576 = 128 x 192, wo_b K = 16384 = 128 x 128):
# 128 heads, 128 + 64 key values, 128 values, one latent row of 512 + 64 a token.
_R, _P, _N, _V = 512, 64, 128, 128


def listed():
    return [
        # The rotation of one decode step's queries: 64 sequences, launch latency.
        {"name": "norm_rope_decode_t64", "op": "norm_rope", "T": 64, "H": 128, "D": 192, "P": 64, "norm": False,
         "weight": False, "inverse": False, "interleaved": True},
        # A long prompt's queries, normalised a head, an odd number of tokens.
        {"name": "norm_rope_prefill_t8191", "op": "norm_rope", "T": 8191, "H": 64, "D": 512, "P": 64, "norm": True,
         "weight": True, "inverse": False, "interleaved": True},
        # One decode step's new rows into an 8-bit cache.
        {"name": "append_e4m3_t32", "op": "append", "T": 32, "R": _R, "P": _P, "page": 64, "pages": 512,
         "dtype": "e4m3", "rows": False, "interleaved": True},
        # A prompt's rows into a bf16 cache; the expanded form reads the rows that come back.
        {"name": "append_bf16_t16381", "op": "append", "T": 16381, "R": _R, "P": _P, "page": 16, "pages": 1200,
         "dtype": "bf16", "rows": True, "interleaved": True},
        # The queries of a decode step into the latent space: weights are read once for few rows.
        {"name": "project_q_t48", "op": "project", "T": 48, "H": 128, "K": _N, "N": _R},
        # The outputs of a prompt chunk back to head values.
        {"name": "project_out_t2047", "op": "project", "T": 2047, "H": 128, "K": _R, "N": _V},
        # One sequence, one token, a tensor-parallel rank's heads, a long context: few rows, one long axis.
        {"name": "absorbed_long_b1", "op": "absorbed", "B": 1, "H": 16, "n": 1, "low": 130000, "high": 131071,
         "R": _R, "P": _P, "page": 64, "dtype": "bf16", "lse": False},
        # A decode batch with all heads on one GPU and contexts of every length.
        {"name": "absorbed_heads128_b64", "op": "absorbed", "B": 64, "H": 128, "n": 1, "low": 1, "high": 8192,
         "R": _R, "P": _P, "page": 64, "dtype": "bf16", "lse": False},
        # A rank's decode batch with two query tokens a sequence over an 8-bit cache of small pages.
        {"name": "absorbed_e4m3_b96", "op": "absorbed", "B": 96, "H": 16, "n": 2, "low": 17, "high": 6000,
         "R": _R, "P": _P, "page": 16, "dtype": "e4m3", "lse": True},
        # Prompts of mixed lengths in one batch, all heads.
        {"name": "expanded_ragged_b7", "op": "expanded", "B": 7, "H": 128, "T": 1111, "past": 0, "N": _N, "P": _P,
         "V": _V, "lse": False},
        # One long prompt on a tensor-parallel rank.
        {"name": "expanded_long_b1", "op": "expanded", "B": 1, "H": 16, "T": 16384, "past": 0, "N": _N, "P": _P,
         "V": _V, "lse": False},
        # A short chunk of a prompt against a long context: few query rows, a long axis.
        {"name": "expanded_chunk_b2", "op": "expanded", "B": 2, "H": 32, "T": 65, "past": 20000, "N": _N, "P": _P,
         "V": _V, "lse": True},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm_rope", "append", "project", "absorbed", "absorbed", "absorbed", "expanded", "expanded"])
    flip = lambda: rng.random() < 0.5  # noqa: E731
    if op == "norm_rope":
        D = rng.choice([64, 128, 192, 192, 512, 576, 2 * rng.randrange(16, 300)])
        H = _log_int(rng, 1, 128)
        T = _log_int(rng, 1, max(1, min(16384, 8191 * 64 * 512 // (H * D))))
        return {"op": op, "T": T, "H": H, "D": D, "P": min(D, rng.choice([32, 64, 64, 128])), "norm": flip(),
                "weight": flip(), "inverse": flip(), "interleaved": flip()}
    if op == "append":
        page = rng.choice([1, 16, 48, 64, 256])
        T = _log_int(rng, 1, 16381)
        return {"op": op, "T": T, "R": rng.choice([512, 512, 256]), "P": rng.choice([64, 64, 0]), "page": page,
                "pages": (T + T // 4 + 512) // page + 2, "dtype": rng.choice(["bf16", "e4m3"]), "rows": flip(),
                "interleaved": flip()}
    if op == "project":
        K, N = rng.choice([(_N, _R), (_R, _V), (_N, _R), (_R, _V), (64, 256), (256, 64),
                           (16 * rng.randrange(4, 32), 16 * rng.randrange(4, 32))])
        H = _log_int(rng, 1, 128)
        T = _log_int(rng, 1, max(1, min(4096, 2047 * 128 * _R * _V // (H * K * N))))
        return {"op": op, "T": T, "H": H, "K": K, "N": N}
    if op == "absorbed":
        H = rng.choice([1, 5, 8, 16, 16, 32, 64, 128, 128])
        B = _log_int(rng, 1, 128)
        n = rng.choice([1, 1, 1, 2, 3, 5])
        most = max(2, min(131071, 64 * 8192 * 128 // (B * H * n), 64 * 8192 // B))
        high = _log_int(rng, 2, most)
        return {"op": op, "B": B, "H": H, "n": n, "low": rng.choice([0, 1, max(1, high // 2)]), "high": high,
                "R": rng.choice([512, 512, 512, 256]), "P": rng.choice([64, 64, 64, 0]),
                "page": rng.choice([1, 16, 48, 64, 128]), "dtype": rng.choice(["bf16", "e4m3"]), "lse": flip()}
    H = rng.choice([1, 4, 16, 16, 32, 128])
    B = _log_int(rng, 1, 12)
    # H * B * T * (T + past) within the long prompt's score matrix of the plain form
    T = _log_int(rng, 1, max(1, min(16384, int(16384 / math.sqrt(max(1.0, B * H / 16))))))
    past = rng.choice([0, 0, rng.randrange(1, 2 + min(32768, max(0, 16 * 16384 * 16384 // (B * H * T) - T)))])
    N, P, V = rng.choice([(_N, _P, _V), (_N, _P, _V), (128, 0, 128), (64, 64, 64), (64, 0, 64)])
    while H * B * T * (T + past) > 16 * 16384 * 16384 or B * (T + past) * H * (N + V) > (1 << 31):
        T, past = max(1, T // 2), past // 2
    return {"op": op, "B": B, "H": H, "T": T, "past": past, "N": N, "P": P, "V": V, "lse": flip()}


# ---- inputs ----------------------------------------------------------------------------------------------------


def _lengths(case, seed):
    """Query and key lengths of a case's sequences: the same ones for every seed, in an order of the seed."""
    import random

    rng = random.Random(seed * 7919 + 13)
    if case["op"] == "absorbed":
        B, low, high = case["B"], case["low"], case["high"]
        kv = [low + (high - low) * (i + 1) // B for i in range(B)]
        rng.shuffle(kv)
        return [case["n"]] * B, kv
    B, T = case["B"], case["T"]
    both = [(max(1, T * (i + 1) // B), case["past"] * (B - i) // B) for i in range(B)]
    rng.shuffle(both)
    return [n for n, _ in both], [n + past for n, past in both]


def _starts(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def _table(P, count, device):
    """cos | sin of every position's angles, taken in 64 bits."""
    inv = 10000.0 ** (-torch.arange(0, P, 2, dtype=torch.float64, device=device) / P)
    a = torch.arange(count, dtype=torch.float64, device=device)[:, None] * inv[None, :]
    return torch.cat([a.cos(), a.sin()], 1).float().contiguous()


def _e4m3(x):
    """Latent rows as 8-bit values and their scale: what an append leaves in the cache."""
    scale = x.float().abs().amax(-1) / _E4M3_MAX
    scale = torch.where(scale > 0, scale, torch.ones_like(scale))
    return (x.float() / scale[..., None]).clamp(-_E4M3_MAX, _E4M3_MAX).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(1000003 * seed + 17)
    op = case["op"]

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=g, device=DEV, dtype=torch.bfloat16) * std

    st = {"case": case}
    if op == "norm_rope":
        T, H, D, P = case["T"], case["H"], case["D"], case["P"]
        st |= {"x": normal(T, H, D, std=2.0), "cos_sin": _table(P, 16384, DEV),
               "pos": torch.randint(0, 16384, (T,), generator=g, device=DEV),
               "weight": 1 + 0.1 * normal(D) if case["norm"] and case["weight"] else None}
    elif op == "append":
        T, R, P, page, pages = case["T"], case["R"], case["P"], case["page"], case["pages"]
        kv = normal(T, R + P, std=1.5)
        kv[:, :8] *= 6  # a few channels of large values, as a latent projection has them
        slots = torch.randperm(page * pages, generator=g, device=DEV)[:T].clone()
        if T > 8:
            slots[T - T // 16 - 1:] = -1  # the padding rows of a captured batch
        st |= {"kv": kv, "slots": slots, "pos": torch.randint(0, 16384, (T,), generator=g, device=DEV),
               "cos_sin": _table(P or 64, 16384, DEV), "weight": 1 + 0.1 * normal(R)}
        dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float8_e4m3fn
        st["latent"] = torch.zeros((pages, page, R), dtype=torch.bfloat16, device=DEV).to(dt)
        st["rope"] = torch.zeros((pages, page, P), dtype=torch.bfloat16, device=DEV).to(dt) if P else None
        st["scale"] = torch.zeros((pages, page), device=DEV) if case["dtype"] == "e4m3" else None
    elif op == "project":
        T, H, K, N = case["T"], case["H"], case["K"], case["N"]
        st |= {"x": normal(T, H, K), "weight": normal(H, N, K, std=K ** -0.5)}
        if own:
            from fused_cpp_amd import latent_attention as la
            st["prepared"] = la.prepare_head_projection(st["weight"])
    elif op == "absorbed":
        B, H, R, P, page = case["B"], case["H"], case["R"], case["P"], case["page"]
        new, kv = _lengths(case, seed)
        width = max(1, max((n + page - 1) // page for n in kv))
        pages = sum((n + page - 1) // page for n in kv) + 1
        order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
        used = torch.tensor([(n + page - 1) // page for n in kv], device=DEV)
        first = torch.cumsum(used, 0) - used
        col = torch.arange(width, device=DEV)[None, :]
        table = torch.where(col < used[:, None], order[(first[:, None] + col).clamp(max=pages - 1)],
                            torch.zeros((), dtype=torch.int32, device=DEV))
        T = sum(new)
        rows = normal(pages, page, R + P)
        scale = None
        if case["dtype"] == "e4m3":
            rows, scale = _e4m3(rows)
        st |= {"q_latent": normal(T, H, R, std=1.5), "q_rope": normal(T, H, P, std=1.5) if P else None,
               "latent": rows[..., :R].contiguous(), "rope": rows[..., R:].contiguous() if P else None,
               "scale": scale, "table": table.contiguous(),
               "lens": torch.tensor(kv, dtype=torch.int32, device=DEV),
               "starts": torch.tensor(_starts(new), dtype=torch.int32, device=DEV),
               "sm": (_N + P) ** -0.5, "n_max": max(new), "kv_max": max(1, max(kv))}
    else:
        H, N, P, V = case["H"], case["N"], case["P"], case["V"]
        new, kv = _lengths(case, seed)
        st |= {"q": normal(sum(new), H, N + P, std=1.5), "kv": normal(sum(kv), H, N + V),
               "k_rope": normal(sum(kv), P) if P else None,
               "starts": torch.tensor(_starts(new), dtype=torch.int32, device=DEV),
               "kv_starts": torch.tensor(_starts(kv), dtype=torch.int32, device=DEV),
               "sm": (N + P) ** -0.5, "n_max": max(new), "kv_max": max(kv)}
    return st


# ---- the framework's calls --------------------------------------------------------------------------------------


def _run_own(st):
    from fused_cpp_amd import latent_attention as la

    case = st["case"]
    op = case["op"]
    if op == "norm_rope":
        return la.head_norm_rope(st["x"], st["pos"], st["cos_sin"], weight=st["weight"], normalize=case["norm"],
                                 inverse=case["inverse"], interleaved=case["interleaved"])
    if op == "append":
        cache = la.LatentCache(st["latent"], st["rope"], st["scale"])
        rows = la.latent_cache_append(st["kv"], st["pos"], st["slots"], st["cos_sin"], cache, weight=st["weight"],
                                      interleaved=case["interleaved"], return_rows=case["rows"])
        return [t for t in (st["latent"], st["rope"], st["scale"], rows) if t is not None]
    if op == "project":
        return la.head_projection(st["x"], st["prepared"])
    if op == "absorbed":
        return la.absorbed_attention(st["q_latent"], st["q_rope"],
                                     la.LatentCache(st["latent"], st["rope"], st["scale"]), st["table"], st["lens"],
                                     scale=st["sm"], query_starts=st["starts"] if case["n"] > 1 else None,
                                     return_lse=case["lse"])
    return la.expanded_attention(st["q"], st["kv"], st["k_rope"], st["starts"], kv_starts=st["kv_starts"],
                                 scale=st["sm"], causal=True, return_lse=case["lse"])


# ---- the plain form ---------------------------------------------------------------------------------------------


def _rotate(x, rows, interleaved, inverse):
    """Rotates the last values of fp32 ``x [T, ..., D]`` by the table rows ``[T, P]`` (cos | sin)."""
    P = rows.shape[1]
    rows = rows.reshape(rows.shape[0], *([1] * (x.dim() - 2)), P)
    cos, sin = rows[..., :P // 2], rows[..., P // 2:]
    sin = -sin if inverse else sin
    keep, r = x[..., :x.shape[-1] - P], x[..., x.shape[-1] - P:]
    if interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = r[..., :P // 2], r[..., P // 2:]
        r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([keep, r], -1)


def _attend(q, k, v, sm, n, kv, n_max, want_lse):
    """Padded fp32 attention: q [G, M, D], k [G, S, D], v [G, S, V]. Row r of a group is query i = r % n_max of its
    ``n``; it sees its keys up to kv - n + i. A row that sees none is 0 with lse -inf."""
    s = torch.bmm(q, k.transpose(1, 2).contiguous()) * sm
    i = (torch.arange(q.shape[1], device=q.device) % n_max)[None, :, None]
    j = torch.arange(k.shape[1], device=q.device)[None, None, :]
    s.masked_fill_(j > (kv - n)[:, None, None] + i, -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    s.sub_(top).exp_()
    total = s.sum(-1, keepdim=True)
    out = torch.bmm(s, v.contiguous()) / torch.where(total > 0, total, torch.ones_like(total))
    return out, (top + total.log())[..., 0] if want_lse else None


def _run_plain(st):
    case = st["case"]
    op = case["op"]
    if op == "norm_rope":
        x = st["x"].float()
        if case["norm"]:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
            if st["weight"] is not None:
                x = x * st["weight"].float()
        return _rotate(x, st["cos_sin"][st["pos"]], case["interleaved"], case["inverse"]).to(torch.bfloat16)
    if op == "append":
        R, P = case["R"], case["P"]
        x = st["kv"].float()
        c = x[:, :R]
        c = c * torch.rsqrt(c.square().mean(-1, keepdim=True) + 1e-6) * st["weight"].float()
        row = _rotate(torch.cat([c, x[:, R:]], 1), st["cos_sin"][st["pos"]], case["interleaved"], False)
        # rows without a slot repeat the first row, which has one: no row is picked out on the host
        kept = torch.where(st["slots"] >= 0, torch.arange(row.shape[0], device=DEV), 0)
        at = st["slots"][kept]
        new = row[kept]
        if case["dtype"] == "e4m3":
            new, scale = _e4m3(new)
            st["scale"].view(-1)[at] = scale
            new = new.view(torch.uint8)
            st["latent"].view(torch.uint8).view(-1, R)[at] = new[:, :R]
            if P:
                st["rope"].view(torch.uint8).view(-1, P)[at] = new[:, R:]
        else:
            new = new.to(torch.bfloat16)
            st["latent"].view(-1, R)[at] = new[:, :R]
            if P:
                st["rope"].view(-1, P)[at] = new[:, R:]
        rows = row.to(torch.bfloat16) if case["rows"] else None
        return [t for t in (st["latent"], st["rope"], st["scale"], rows) if t is not None]
    if op == "project":
        x, w = st["x"].float().transpose(0, 1).contiguous(), st["weight"].float().transpose(1, 2).contiguous()
        return torch.bmm(x, w).transpose(0, 1).to(torch.bfloat16).contiguous()

    starts = st["starts"].long()
    n = starts[1:] - starts[:-1]
    row = torch.arange(st["n_max"], device=DEV)[None, :]
    at = (starts[:-1, None] + row).clamp(max=int(st["q_latent" if op == "absorbed" else "q"].shape[0]) - 1)  # [B, n]
    token = torch.arange(int(st["q_latent" if op == "absorbed" else "q"].shape[0]), device=DEV)
    seq = torch.searchsorted(starts[1:].contiguous(), token, right=True)
    back = lambda x: x.transpose(1, 2)[seq, token - starts[seq]]  # noqa: E731  [B, H, n, ...] -> [T, H, ...]
    col = torch.arange(st["kv_max"], device=DEV)
    if op == "absorbed":
        B, H, R, P, page = case["B"], case["H"], case["R"], case["P"], case["page"]
        slot = st["table"].long()[:, col // page] * page + col % page  # [B, S]
        k = st["latent"].view(-1, R)[slot].float()
        q = st["q_latent"].float()
        if P:
            k = torch.cat([k, st["rope"].view(-1, P)[slot].float()], -1)
            q = torch.cat([q, st["q_rope"].float()], -1)
        if st["scale"] is not None:
            k = k * st["scale"].view(-1)[slot][..., None]
        q = q[at]  # [B, n, H, R + P]
        # the heads of a sequence share its keys: one group holds the rows of all its heads
        q = q.transpose(1, 2).reshape(B, H * st["n_max"], R + P)
        out, lse = _attend(q, k, k[..., :R], st["sm"], n, st["lens"].long(), st["n_max"], case["lse"])
        out = back(out.view(B, H, st["n_max"], R)).to(torch.bfloat16)
        return (out, back(lse.view(B, H, st["n_max"]))) if case["lse"] else out
    H, N, P, V = case["H"], case["N"], case["P"], case["V"]
    B = case["B"]
    kvs = st["kv_starts"].long()
    at_k = (kvs[:-1, None] + col[None, :]).clamp(max=int(st["kv"].shape[0]) - 1)
    kv = st["kv"].float()
    k, v = kv[..., :N], kv[..., N:]
    if P:
        k = torch.cat([k, st["k_rope"].float()[:, None, :].expand(-1, H, -1)], -1)
    heads = lambda x, i: x[i].transpose(1, 2).reshape(B * H, i.shape[1], x.shape[-1])  # noqa: E731
    out, lse = _attend(heads(st["q"].float(), at), heads(k, at_k), heads(v, at_k), st["sm"],
                       n.repeat_interleave(H), (kvs[1:] - kvs[:-1]).repeat_interleave(H), st["n_max"], case["lse"])
    out = back(out.view(B, H, st["n_max"], V)).to(torch.bfloat16)
    return (out, back(lse.view(B, H, st["n_max"]))) if case["lse"] else out


def run(state):
    if own:
        return _run_own(state)
    return _run_plain(state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------


def _visible(new, kv):
    """Query-key pairs of a causal batch."""
    return sum(sum(max(0, min(L, L - n + i + 1)) for i in range(n)) if n < 64 else
               n * (L - n) + n * (n + 1) // 2 if L >= n else L * (L + 1) // 2 for n, L in zip(new, kv))


def work(case):
    op = case["op"]
    if op == "norm_rope":
        e = case["T"] * case["H"] * case["D"]
        return {"bytes": 4 * e + case["T"] * (4 * case["P"] + 8), "flops": (5 if case["norm"] else 0) * e
                + 3 * case["T"] * case["H"] * case["P"]}
    if op == "append":
        T, W = case["T"], case["R"] + case["P"]
        kept = T - (T // 16 + 1 if T > 8 else 0)
        size = 2 if case["dtype"] == "bf16" else 1
        # rows that no output holds are not read
        read = T if case["rows"] else kept
        return {"bytes": read * (2 * W + 16 + 4 * (case["P"] or 64)) + kept * (size * W + (4 if size == 1 else 0))
                + (2 * T * W if case["rows"] else 0), "flops": 6 * read * W}
    if op == "project":
        T, H, K, N = case["T"], case["H"], case["K"], case["N"]
        return {"bytes": 2 * H * N * K + 2 * T * H * (K + N), "flops": 2 * T * H * K * N}
    new, kv = _lengths(case, 0)
    if op == "absorbed":
        H, R, P = case["H"], case["R"], case["P"]
        row = 2 * (R + P) if case["dtype"] == "bf16" else R + P + 4
        return {"bytes": sum(kv) * row + 2 * sum(new) * H * (2 * R + P) + (4 * sum(new) * H if case["lse"] else 0),
                "flops": 2 * H * _visible(new, kv) * (2 * R + P)}
    H, N, P, V = case["H"], case["N"], case["P"], case["V"]
    return {"bytes": 2 * sum(new) * H * (N + P + V) + 2 * sum(kv) * (H * (N + V) + P)
            + (4 * sum(new) * H if case["lse"] else 0), "flops": 2 * H * _visible(new, kv) * (N + P + V)}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------


def _turned(vec, angles_row, interleaved, sign):
    """One tensor of rows [T, H, D] as complex numbers times exp(i * sign * angle): the rotation's definition."""
    P = angles_row.shape[-1]
    turn = torch.complex(angles_row[:, :P // 2], sign * angles_row[:, P // 2:])[:, None, :]
    tail = vec[:, :, vec.shape[2] - P:]
    if interleaved:
        z = torch.view_as_complex(tail.unflatten(-1, (P // 2, 2)).contiguous()) * turn
        tail = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(tail[:, :, :P // 2].contiguous(), tail[:, :, P // 2:].contiguous()) * turn
        tail = torch.cat([z.real, z.imag], -1)
    out = vec.clone()
    out[:, :, vec.shape[2] - P:] = tail
    return out


def exact(case, seed):
    op = case["op"]
    st = prepare(case, seed)
    f64 = torch.float64
    if op == "norm_rope":
        vec = st["x"].to(f64)
        if case["norm"]:
            vec = vec / (vec.pow(2).sum(-1, keepdim=True) / case["D"] + 1e-6).sqrt()
            vec = vec if st["weight"] is None else vec * st["weight"].to(f64)
        return _turned(vec, st["cos_sin"].to(f64)[st["pos"]], case["interleaved"], -1.0 if case["inverse"] else 1.0)
    if op == "append":
        R, P = case["R"], case["P"]
        vec = st["kv"].to(f64)
        vec[:, :R] = vec[:, :R] / (vec[:, :R].pow(2).sum(-1, keepdim=True) / R + 1e-6).sqrt() * st["weight"].to(f64)
        vec = _turned(vec[:, None, :], st["cos_sin"].to(f64)[st["pos"]], case["interleaved"], 1.0)[:, 0]
        out = torch.zeros((case["pages"] * case["page"], R + P), dtype=f64, device=DEV)
        who = torch.nonzero(st["slots"] >= 0)[:, 0]
        scales = None
        if case["dtype"] == "e4m3":
            scales = torch.zeros((out.shape[0],), dtype=f64, device=DEV)
            scales[st["slots"][who]] = vec[who].abs().amax(1) / _E4M3_MAX
            out[st["slots"][who]] = vec[who] / scales[st["slots"][who]][:, None]
            scales = scales.view(case["pages"], case["page"])
        else:
            out[st["slots"][who]] = vec[who]
        out = out.view(case["pages"], case["page"], R + P)
        return [t for t in (out[..., :R], out[..., R:] if P else None, scales, vec if case["rows"] else None)
                if t is not None]
    if op == "project":
        out = torch.empty((case["T"], case["H"], case["N"]), dtype=f64, device=DEV)
        for h in range(case["H"]):
            out[:, h] = st["x"][:, h].to(f64) @ st["weight"][h].to(f64).T.contiguous()
        return out
    if work(case)["flops"] > 2e12:
        return None
    new, kv = _lengths(case, seed)
    outs, lses = [], []
    first_q = first_k = 0
    for b, (n, L) in enumerate(zip(new, kv)):
        keep = torch.arange(L, device=DEV)[None, :] <= (L - n) + torch.arange(n, device=DEV)[:, None]
        per = []
        if op == "absorbed":
            R, P, page = case["R"], case["P"], case["page"]
            use = (L + page - 1) // page
            ids = st["table"][b, :use].long()
            rows = st["latent"][ids].reshape(use * page, R)[:L].to(f64)
            if P:
                rows = torch.cat([rows, st["rope"][ids].reshape(use * page, P)[:L].to(f64)], 1)
            if st["scale"] is not None:
                rows = rows * st["scale"][ids].reshape(use * page)[:L, None].to(f64)
            keys_t = rows.T.contiguous()
        for h in range(case["H"]):
            if op == "absorbed":
                q = st["q_latent"][first_q:first_q + n, h].to(f64)
                if P:
                    q = torch.cat([q, st["q_rope"][first_q:first_q + n, h].to(f64)], 1)
                values = rows[:, :R]
            else:
                N = case["N"]
                q = st["q"][first_q:first_q + n, h].to(f64)
                mine = st["kv"][first_k:first_k + L, h].to(f64)
                keys_t = mine[:, :N]
                if case["P"]:
                    keys_t = torch.cat([keys_t, st["k_rope"][first_k:first_k + L].to(f64)], 1)
                keys_t = keys_t.T.contiguous()
                values = mine[:, N:].contiguous()
            s = (q @ keys_t) * st["sm"]
            s = torch.where(keep, s, torch.full_like(s, -math.inf))
            lse = torch.logsumexp(s, 1)
            p = torch.where(keep, (s - torch.where(lse == -math.inf, torch.zeros_like(lse), lse)[:, None]).exp(),
                            torch.zeros_like(s))
            per.append((p @ values, lse))
        outs.append(torch.stack([o for o, _ in per], 1))
        lses.append(torch.stack([x for _, x in per], 1))
        first_q += n
        first_k += L
    out = torch.cat(outs, 0)
    return (out, torch.cat(lses, 0)) if case["lse"] else out
