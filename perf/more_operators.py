"""The measured work of ``fused_cpp_amd.latent_attention`` beyond plain causal attention and of
``fused_cpp_amd.latent_context``: what serving long contexts and drafted tokens over a latent cache needs, each through
its public entry point.

A case is a dict of plain values with an ``op``:

* ``window``: absorbed attention of ``n`` query tokens a sequence that see their last ``window`` tokens and the first
  ``sinks`` of the sequence.
* ``prompt``: expanded attention of ``B`` sequences of up to ``T`` new tokens behind up to ``past`` earlier ones, with
  the same window and first tokens.
* ``tree``: absorbed attention of a tree of up to ``nodes`` drafted tokens a sequence, from its parents.
* ``weights``: what each cached token received of the softmax weights of ``n`` query tokens' heads, added to what it
  had.
* ``heaviest``: the positions that stay when a sequence keeps ``keep`` tokens (its first, its last, and the heaviest),
  and their weights.
* ``move``: cached rows to other rows: an eviction's kept rows into fresh pages, accepted drafts behind their context.

``own`` picks the framework's kernels; without it ``run`` computes the operators from elementary operations in
32 bits.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
_E4M3_MAX = 448.0

# The layer that the repository's W8A8 projections belong to: 128 heads, 128 + 64 key values, 128 values, one latent
# row of 512 + 64 a token.
_R, _P, _N, _V = 512, 64, 128, 128


def listed():
    return [
        # One sequence, one token, a tensor-parallel rank's heads: a long context cut to a window, latency.
        {"name": "window_b1", "op": "window", "B": 1, "H": 16, "n": 1, "low": 130000, "high": 131071, "window": 4096,
         "sinks": 4, "R": _R, "P": _P, "page": 64, "dtype": "bf16", "lse": False},
        # A decode batch with all heads, two query tokens a sequence, an 8-bit cache of small pages.
        {"name": "window_e4m3_b96", "op": "window", "B": 96, "H": 128, "n": 2, "low": 1, "high": 8192, "window": 1000,
         "sinks": 64, "R": _R, "P": _P, "page": 16, "dtype": "e4m3", "lse": True},
        # One long prompt on a rank.
        {"name": "prompt_b1", "op": "prompt", "B": 1, "H": 16, "T": 16384, "past": 0, "window": 1024, "sinks": 4,
         "N": _N, "P": _P, "V": _V, "lse": False},
        # Chunks of prompts of several lengths behind long contexts.
        {"name": "prompt_chunk_b5", "op": "prompt", "B": 5, "H": 32, "T": 333, "past": 20000, "window": 2048,
         "sinks": 64, "N": _N, "P": _P, "V": _V, "lse": True},
        # One user's wide tree behind a long context, a rank's heads.
        {"name": "tree_b1", "op": "tree", "B": 1, "H": 16, "nodes": 60, "low": 31000, "high": 32000, "R": _R, "P": _P,
         "page": 64, "dtype": "bf16", "lse": False},
        # A batch of small trees, all heads, an 8-bit cache of small pages.
        {"name": "tree_e4m3_b32", "op": "tree", "B": 32, "H": 128, "nodes": 9, "low": 1, "high": 8192, "R": _R,
         "P": _P, "page": 16, "dtype": "e4m3", "lse": True},
        # A decode step of a batch that counts its heavy tokens, a rank's heads.
        {"name": "weights_b64", "op": "weights", "B": 64, "H": 16, "n": 1, "low": 1, "high": 8192, "R": _R, "P": _P,
         "page": 64, "dtype": "bf16"},
        # The last tokens of two prompts, all heads: what an eviction after the prompts goes by.
        {"name": "weights_prompt_b2", "op": "weights", "B": 2, "H": 128, "n": 32, "low": 16000, "high": 16384, "R": _R,
         "P": _P, "page": 16, "dtype": "bf16"},
        # One long context cut down once.
        {"name": "heaviest_b1", "op": "heaviest", "B": 1, "low": 131000, "high": 131071, "keep": 4096, "sinks": 4,
         "recent": 64},
        # A batch of contexts of every length; the shorter ones keep all they have.
        {"name": "heaviest_b64", "op": "heaviest", "B": 64, "low": 1, "high": 8192, "keep": 2048, "sinks": 4,
         "recent": 128},
        # The accepted drafts of a batch behind their contexts: a few rows a sequence, latency.
        {"name": "move_drafts_b32", "op": "move", "B": 32, "low": 100, "high": 8192, "keep": 5, "R": _R, "P": _P,
         "page": 64, "dtype": "bf16", "drafts": True},
        # An eviction's kept rows into fresh pages.
        {"name": "move_kept_b64", "op": "move", "B": 64, "low": 1, "high": 8192, "keep": 2048, "R": _R, "P": _P,
         "page": 16, "dtype": "bf16", "drafts": False},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["window", "window", "prompt", "prompt", "tree", "tree", "weights", "heaviest", "move"])
    flip = lambda: rng.random() < 0.5  # noqa: E731
    cache = {"R": rng.choice([512, 512, 512, 256]), "P": rng.choice([64, 64, 64, 0]),
             "page": rng.choice([1, 16, 48, 64, 128]), "dtype": rng.choice(["bf16", "e4m3"])}
    if op == "window":
        H, B, n = rng.choice([1, 5, 8, 16, 16, 32, 128, 128]), _log_int(rng, 1, 96), rng.choice([1, 1, 1, 2, 3, 5])
        high = _log_int(rng, 2, min(131071, 96 * 8192 // B))
        window = _log_int(rng, 1, max(2, min(8192, 96 * 2 * 128 * 1000 // (B * n * H))))
        return {"op": op, "B": B, "H": H, "n": n, "low": rng.choice([0, 1, max(1, high // 2)]), "high": high,
                "window": window, "sinks": rng.choice([0, 1, 4, 64, 130]), **cache, "lse": flip()}
    if op == "prompt":
        H, B = rng.choice([1, 4, 16, 16, 32]), _log_int(rng, 1, 12)
        T = _log_int(rng, 1, max(1, 16384 * 16 // (B * H) if H > 16 else 16384 // B))
        past = rng.choice([0, 0, rng.randrange(1, max(2, 100000 // (B * H)))])
        window = _log_int(rng, 1, max(2, min(8192, 16 * 16384 * 1024 // (H * B * T))))
        N, P, V = rng.choice([(_N, _P, _V), (_N, _P, _V), (128, 0, 128), (64, 64, 64), (64, 0, 64)])
        return {"op": op, "B": B, "H": H, "T": T, "past": past, "window": window,
                "sinks": rng.choice([0, 1, 4, 64, 130]), "N": N, "P": P, "V": V, "lse": flip()}
    if op == "tree":
        H, B, nodes = rng.choice([1, 5, 8, 16, 16, 32, 128]), _log_int(rng, 1, 64), _log_int(rng, 1, 200)
        nodes = max(1, min(nodes, 8 * 8192 // (B * H)))
        high = _log_int(rng, 2, max(2, min(32000, 32 * 9 * 128 * 7000 // (2 * B * H * nodes), 16 * 8192 // B)))
        return {"op": op, "B": B, "H": H, "nodes": nodes, "low": rng.choice([0, 1, max(1, high // 2)]), "high": high,
                **cache, "lse": flip()}
    if op == "weights":
        H, B, n = rng.choice([1, 5, 8, 16, 16, 32, 128]), _log_int(rng, 1, 64), _log_int(rng, 1, 48)
        n = max(1, min(n, 2 * 128 * 32 // (B * H)))
        high = _log_int(rng, 2, max(2, min(131071, 48 * 8192 // B, 2 * 128 * 32 * 16384 // (B * H * n))))
        return {"op": op, "B": B, "H": H, "n": n, "low": rng.choice([0, 1, max(1, high // 2)]), "high": high, **cache}
    B = _log_int(rng, 1, 64)
    high = _log_int(rng, 2, min(131071, 64 * 8192 // B))
    low = rng.choice([0, 1, max(1, high // 2)])
    if op == "heaviest":
        keep = _log_int(rng, 1, max(2, min(8192, high)))
        sinks = rng.choice([0, 1, 4, 64])
        recent = rng.randrange(0, 1 + max(0, keep - min(sinks, keep)))
        return {"op": op, "B": B, "low": low, "high": high, "keep": keep, "sinks": min(sinks, keep), "recent": recent}
    drafts = flip()
    keep = _log_int(rng, 1, 16) if drafts else _log_int(rng, 1, max(2, min(2048 * 64 // B, high)))
    return {"op": op, "B": B, "low": low, "high": high, "keep": keep, **cache, "drafts": drafts}


# ---- inputs ----------------------------------------------------------------------------------------------------


def _lengths(case, seed):
    """New tokens and all tokens of a case's sequences: the same ones for every seed, in an order of the seed."""
    rng = random.Random(seed * 7919 + 13)
    B = case["B"]
    if case["op"] == "prompt":
        both = [(max(1, case["T"] * (i + 1) // B), case["past"] * (B - i) // B) for i in range(B)]
        rng.shuffle(both)
        return [n for n, _ in both], [n + past for n, past in both]
    kv = [case["low"] + (case["high"] - case["low"]) * (i + 1) // B for i in range(B)]
    rng.shuffle(kv)
    if case["op"] == "tree":
        new = [max(1, case["nodes"] * (i + 1) // B) for i in range(B)]
        rng.shuffle(new)
        return new, [n + L for n, L in zip(new, kv)]
    return [case.get("n", 1)] * B, kv


def _starts(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def _parents(new, seed):
    """Trees as beams draft them: node i hangs on one of the last few nodes of its sequence, or begins a new branch."""
    rng = random.Random(seed * 104729 + 5)
    out = []
    for n in new:
        out += [rng.choice([-1, -1, i - 1, rng.randrange(max(0, i - 8), i), rng.randrange(i)]) if i else -1
                for i in range(n)]
    return out


def _table(lengths, page, order):
    """Pages of sequences of these lengths, taken in turn from ``order``."""
    used = torch.tensor([(n + page - 1) // page for n in lengths], device=DEV)
    width = max(1, max((n + page - 1) // page for n in lengths))
    first = torch.cumsum(used, 0) - used
    col = torch.arange(width, device=DEV)[None, :]
    at = (first[:, None] + col).clamp(max=order.numel() - 1)
    return torch.where(col < used[:, None], order[at], torch.zeros_like(order[:1])).contiguous()


def _e4m3(x):
    """Latent rows as 8-bit values and their scale: what an append leaves in the cache."""
    scale = x.float().abs().amax(-1) / _E4M3_MAX
    scale = torch.where(scale > 0, scale, torch.ones_like(scale))
    return (x.float() / scale[..., None]).clamp(-_E4M3_MAX, _E4M3_MAX).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(1000003 * seed + 29)
    op = case["op"]

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=g, device=DEV, dtype=torch.bfloat16) * std

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=DEV)

    new, kv = _lengths(case, seed)
    st = {"case": case, "new": new, "kv_lens": kv, "lens": ints(kv)}
    if op == "heaviest":
        # weights as they build up: few heavy tokens, many light ones, some that were never looked at
        w = torch.randn((case["B"], max(1, case["high"])), generator=g, device=DEV).mul_(2.0).exp_()
        w[torch.rand(w.shape, generator=g, device=DEV) < 0.1] = 0.0
        st["weights"] = w
        return st
    if op == "prompt":
        H, N, P, V = case["H"], case["N"], case["P"], case["V"]
        st |= {"q": normal(sum(new), H, N + P, std=1.5), "kv": normal(sum(kv), H, N + V),
               "k_rope": normal(sum(kv), P) if P else None, "starts": ints(_starts(new)),
               "kv_starts": ints(_starts(kv)), "sm": (N + P) ** -0.5}
        return st
    B, R, P, page = case["B"], case["R"], case["P"], case["page"]
    rest = 0
    if op == "move":
        kept = [min(case["keep"], max(1, n)) if not case["drafts"] else case["keep"] for n in kv]
        rest = sum((n + page - 1) // page + 1 for n in (k + (L if case["drafts"] else 0) for k, L in zip(kept, kv)))
    pages = sum((n + page - 1) // page for n in kv) + rest + 1
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    st["table"] = _table(kv, page, order)
    rows = normal(pages, page, R + P)
    scale = None
    if case["dtype"] == "e4m3":
        rows, scale = _e4m3(rows)
    st |= {"latent": rows[..., :R].contiguous(), "rope": rows[..., R:].contiguous() if P else None, "scale": scale}
    if op == "move":
        behind = order[sum((n + page - 1) // page for n in kv):]
        m = max(kept)
        pos, counts, first, to = [], [], [], []
        rng = random.Random(seed * 31 + 7)
        for k, L in zip(kept, kv):
            k = min(k, L)
            if case["drafts"]:  # some of the last rows, to be continued elsewhere behind as many
                k = rng.randrange(k + 1)
                low = max(0, L - 4 * case["keep"])
                chosen = sorted(rng.sample(range(low, L), k)) if k else []
                first.append(low)
                to.append(low + case["keep"])
            else:
                chosen = None
                first.append(0)
                to.append(max(1, k))
            pos.append(chosen)
            counts.append(k)
        if not case["drafts"]:
            # kept rows anywhere in their sequences, ascending
            r = torch.rand((B, max(1, max(kv))), generator=g, device=DEV)
            r[torch.arange(r.shape[1], device=DEV)[None, :] >= st["lens"][:, None]] = 2.0
            top = r.argsort(1)[:, :m]
            here = torch.arange(top.shape[1], device=DEV)[None, :] < ints(counts)[:, None]
            positions = torch.where(here, top, 1 << 30).sort(1).values
            positions = torch.where(here, positions, -1).to(torch.int32)
        else:
            positions = ints([p + [-1] * (m - len(p)) for p in pos])
        st |= {"positions": positions.contiguous(), "counts": ints(counts), "first": ints(first),
               "to_table": _table(to, page, behind)}
        return st
    T, H = sum(new), case["H"]
    st |= {"q_latent": normal(T, H, R, std=1.5), "q_rope": normal(T, H, P, std=1.5) if P else None,
           "starts": ints(_starts(new)), "sm": (_N + P) ** -0.5}
    if op == "tree":
        st["parents"] = ints(_parents(new, seed))
    if op == "weights":
        st["previous"] = torch.rand((B, max(1, max(kv))), generator=g, device=DEV) * 4
        # the attention's own sums, which the call is given
        lse = torch.empty((T, H), device=DEV)
        for b, (n, L) in enumerate(zip(new, kv)):
            at = torch.arange(L, device=DEV)
            s = _queries(st, b * n, b * n + n).reshape(n * H, -1) @ _rows(st, b, at).T.contiguous() * st["sm"]
            s.masked_fill_(~_seen_by(L - n, L, L + 1, 0, at).repeat_interleave(H, 0), -math.inf)
            lse[b * n:b * n + n] = s.logsumexp(-1).view(n, H)
        st["lse"] = lse
    return st


# ---- the framework's calls --------------------------------------------------------------------------------------


def _run_own(st):
    from fused_cpp_amd import latent_attention as la
    from fused_cpp_amd import latent_context as lc

    case = st["case"]
    op = case["op"]
    if op == "prompt":
        return la.expanded_attention(st["q"], st["kv"], st["k_rope"], st["starts"], kv_starts=st["kv_starts"],
                                     scale=st["sm"], window=case["window"], sinks=case["sinks"],
                                     return_lse=case["lse"])
    if op == "heaviest":
        return lc.heaviest_positions(st["weights"], st["lens"], case["keep"], sinks=case["sinks"],
                                     recent=case["recent"])
    cache = la.LatentCache(st["latent"], st["rope"], st["scale"])
    if op == "window":
        return la.absorbed_attention(st["q_latent"], st["q_rope"], cache, st["table"], st["lens"], scale=st["sm"],
                                     query_starts=st["starts"] if case["n"] > 1 else None, window=case["window"],
                                     sinks=case["sinks"], return_lse=case["lse"])
    if op == "tree":
        tree = lc.draft_tree(st["parents"], st["starts"], case["nodes"])
        got = la.absorbed_attention(st["q_latent"], st["q_rope"], cache, st["table"], st["lens"], scale=st["sm"],
                                    query_starts=st["starts"], tree=tree, return_lse=case["lse"])
        return (*(got if case["lse"] else (got,)), tree.masks, tree.depths)
    if op == "weights":
        return lc.attention_weights(st["q_latent"], st["q_rope"], cache, st["table"], st["lens"], st["lse"],
                                    scale=st["sm"], query_starts=st["starts"] if case["n"] > 1 else None,
                                    previous=st["previous"])
    lc.latent_cache_move(cache, st["table"], st["positions"], st["counts"], to_table=st["to_table"],
                         starts=st["first"] if case["drafts"] else None)
    return [t for t in (st["latent"], st["rope"], st["scale"]) if t is not None]


# ---- the plain form ---------------------------------------------------------------------------------------------


def _rows(st, b, at):
    """Cached rows of sequence b at positions ``at`` in fp32."""
    page, R = st["case"]["page"], st["case"]["R"]
    slot = st["table"][b].long()[at // page] * page + at % page
    k = st["latent"].view(-1, R)[slot].float()
    if st["rope"] is not None:
        k = torch.cat([k, st["rope"].view(-1, st["case"]["P"])[slot].float()], -1)
    return k if st["scale"] is None else k * st["scale"].view(-1)[slot][:, None]


def _queries(st, lo, hi):
    q = st["q_latent"][lo:hi].float()
    return q if st["q_rope"] is None else torch.cat([q, st["q_rope"][lo:hi].float()], -1)


def _softmax(s, keep, v):
    """fp32 scores and what each row sees of them (``keep``), values; a row that sees none is 0 with lse -inf."""
    s = s.masked_fill(~keep, -math.inf)
    top = s.amax(-1, keepdim=True) if s.shape[-1] else s.new_full((*s.shape[:-1], 1), -math.inf)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = (s - top).exp()
    total = e.sum(-1, keepdim=True)
    out = e @ v / torch.where(total > 0, total, torch.ones_like(total))
    return out, (top + total.log())[..., 0]


def _seen_by(lo, hi, window, sinks, at):
    """Rows of positions lo .. hi, keys at positions ``at``: the window behind each row, and the first keys."""
    pos = torch.arange(lo, hi, device=DEV)[:, None]
    return (at[None, :] <= pos) & ((at[None, :] > pos - window) | (at[None, :] < sinks))


def _cut(lo, hi, window, sinks):
    """Key positions that some row of positions lo .. hi sees."""
    first = max(0, lo - window + 1)
    head = torch.arange(min(sinks, first, max(0, hi)), device=DEV)
    return torch.cat([head, torch.arange(first, max(first, hi), device=DEV)])


def _run_plain(st):
    case = st["case"]
    op = case["op"]
    new, kv = st["new"], st["kv_lens"]
    if op == "heaviest":
        keep, sinks, recent = case["keep"], case["sinks"], case["recent"]
        w, lens = st["weights"], st["lens"].long()[:, None]
        at = torch.arange(w.shape[1], device=DEV)[None, :]
        always = (at < sinks) | (at >= lens - recent)
        w = torch.where(at >= lens, -math.inf, torch.where(always, math.inf, w))
        order = w.sort(dim=1, descending=True, stable=True).indices[:, :keep]
        if order.shape[1] < keep:
            order = torch.nn.functional.pad(order, (0, keep - order.shape[1]))
        counts = lens.clamp(max=keep)
        here = torch.arange(keep, device=DEV)[None, :] < counts
        positions = torch.where(here, order, 1 << 40).sort(1).values
        kept = torch.where(here, st["weights"].gather(1, positions.clamp(max=w.shape[1] - 1)), 0.0)
        return torch.where(here, positions, -1).to(torch.int32), counts[:, 0].to(torch.int32), kept
    if op == "move":
        R, P, page = case["R"], case["P"], case["page"]
        k = torch.arange(st["positions"].shape[1], device=DEV)[None, :]
        here = k < st["counts"][:, None]
        source = st["positions"].long().clamp(min=0)
        target = k + st["first"].long()[:, None] if case["drafts"] else k.expand_as(source)
        slots = []
        for table, at in ((st["table"], source), (st["to_table"], target)):
            inside = (at // page).clamp(max=table.shape[1] - 1)
            slots.append(table.long().gather(1, inside) * page + at % page)
        a, b = slots[0][here], slots[1][here]
        for t, width in ((st["latent"], R), (st["rope"], P), (st["scale"], 1)):
            if t is not None:
                flat = (t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t).view(-1, width)
                flat[b] = flat[a]
        return [t for t in (st["latent"], st["rope"], st["scale"]) if t is not None]
    if op == "prompt":
        H, N, P = case["H"], case["N"], case["P"]
        out = torch.empty((sum(new), H, case["V"]), dtype=torch.bfloat16, device=DEV)
        lse = torch.empty((sum(new), H), device=DEV)
        q0 = k0 = 0
        for n, L in zip(new, kv):
            for i in range(0, n, 1024):
                rows = min(1024, n - i)
                lo = L - n + i
                at = _cut(lo, lo + rows, case["window"], case["sinks"])
                both = st["kv"][k0:k0 + L][at].float()
                k = both[..., :N]
                if P:
                    k = torch.cat([k, st["k_rope"][k0:k0 + L][at].float()[:, None, :].expand(-1, H, -1)], -1)
                q = st["q"][q0 + i:q0 + i + rows].float().transpose(0, 1).contiguous()
                s = torch.bmm(q, k.permute(1, 2, 0).contiguous()) * st["sm"]
                o, e = _softmax(s, _seen_by(lo, lo + rows, case["window"], case["sinks"], at)[None],
                                both[..., N:].transpose(0, 1).contiguous())
                out[q0 + i:q0 + i + rows] = o.transpose(0, 1).to(torch.bfloat16)
                lse[q0 + i:q0 + i + rows] = e.T
            q0, k0 = q0 + n, k0 + L
        return (out, lse) if case["lse"] else out
    T, H, R = sum(new), case["H"], case["R"]
    if op == "weights":
        total = st["previous"].clone()
        for b, (n, L) in enumerate(zip(new, kv)):
            k = _rows(st, b, torch.arange(L, device=DEV))
            q = _queries(st, b * n, b * n + n).reshape(n * H, -1)
            p = (q @ k.T.contiguous() * st["sm"] - st["lse"][b * n:b * n + n].reshape(-1, 1)).exp()
            keep = _seen_by(L - n, L, L + 1, 0, torch.arange(L, device=DEV)).repeat_interleave(H, 0)
            total[b, :L] += torch.where(keep, p, torch.zeros_like(p)).sum(0)
        return total
    out = torch.empty((T, H, R), dtype=torch.bfloat16, device=DEV)
    lse = torch.empty((T, H), device=DEV)
    masks = torch.zeros((T, (case.get("nodes", 0) + 63) // 64), dtype=torch.int64, device=DEV)
    depths = torch.zeros((T,), dtype=torch.int32, device=DEV)
    q0 = 0
    for b, (n, L) in enumerate(zip(new, kv)):
        if op == "window":
            at = _cut(L - n, L, case["window"], case["sinks"])
            keep = _seen_by(L - n, L, case["window"], case["sinks"], at)
        else:
            at = torch.arange(L, device=DEV)
            parent = st["parents"][q0:q0 + n].long()
            step = (parent[:, None] == torch.arange(n, device=DEV)[None, :]).float()
            line = torch.eye(n, device=DEV)
            for _ in range(max(1, (n - 1).bit_length())):  # ancestors of 1, 3, 7 .. generations
                line = ((line + step @ line) > 0).float()
                step = ((step @ step) > 0).float()
            line = line > 0
            keep = torch.cat([torch.ones((n, L - n), dtype=torch.bool, device=DEV), line], 1)
            bit = torch.ones((), dtype=torch.int64, device=DEV) << (torch.arange(n, device=DEV) % 64)
            for w in range((n + 63) // 64):
                masks[q0:q0 + n, w] = torch.where(line, bit, 0)[:, 64 * w:64 * w + 64].sum(1)
            depths[q0:q0 + n] = line.sum(1) - 1
        k = _rows(st, b, at)
        q = _queries(st, q0, q0 + n).reshape(n * H, -1)
        o, e = _softmax(q @ k.T.contiguous() * st["sm"], keep.repeat_interleave(H, 0), k[:, :R].contiguous())
        out[q0:q0 + n], lse[q0:q0 + n] = o.view(n, H, R).to(torch.bfloat16), e.view(n, H)
        q0 += n
    got = (out, lse) if case["lse"] else (out,)
    return got if op == "window" and case["lse"] else out if op == "window" else (*got, masks, depths)


def run(state):
    if own:
        return _run_own(state)
    return _run_plain(state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------


def _pairs(n, L, window, sinks):
    """Query-key pairs and keys read of the last n of L tokens."""
    pairs = sum(min(p + 1, window) + max(0, min(sinks, p - window + 1)) for p in range(max(0, L - n), L))
    first = max(0, L - n - window + 1)
    return pairs, L - first + min(sinks, first)


def work(case):
    op = case["op"]
    new, kv = _lengths(case, 0)
    if op == "heaviest":
        low = [L for L in kv if L > case["keep"]]
        read = sum(L - case["sinks"] - case["recent"] for L in low)
        return {"bytes": 4 * read + 8 * case["B"] * (case["keep"] + 1), "flops": read}
    if op == "prompt":
        H, N, P, V = case["H"], case["N"], case["P"], case["V"]
        pairs, keys = map(sum, zip(*(_pairs(n, L, case["window"], case["sinks"]) for n, L in zip(new, kv))))
        return {"bytes": 2 * sum(new) * H * (N + P + V) + 2 * keys * (H * (N + V) + P)
                + (4 * sum(new) * H if case["lse"] else 0), "flops": 2 * H * pairs * (N + P + V)}
    R, P = case["R"], case["P"]
    row = 2 * (R + P) if case["dtype"] == "bf16" else R + P + 4
    if op == "move":
        rows = case["B"] * case["keep"] // 2 if case["drafts"] else sum(min(case["keep"], L) for L in kv)
        return {"bytes": 2 * rows * row + 4 * rows, "flops": 0}
    H, T = case["H"], sum(new)
    if op == "weights":
        pairs = sum(_pairs(n, L, L + 1, 0)[0] for n, L in zip(new, kv))
        return {"bytes": sum(kv) * row + 2 * T * H * (R + P) + 4 * T * H + 8 * case["B"] * max(1, max(kv)),
                "flops": 2 * H * pairs * (R + P)}
    if op == "window":
        pairs, keys = map(sum, zip(*(_pairs(n, L, case["window"], case["sinks"]) for n, L in zip(new, kv))))
    else:
        # a node sees its ancestors among the nodes: few beside the context
        keys, pairs = sum(kv), sum(n * (L - n) + n for n, L in zip(new, kv))
    return {"bytes": keys * row + 2 * T * H * (2 * R + P) + (4 * T * H if case["lse"] else 0),
            "flops": 2 * H * pairs * (2 * R + P)}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------


def exact(case, seed):
    op = case["op"]
    if op == "heaviest":
        st = prepare(case, seed)
        kept = torch.zeros((case["B"], case["keep"]), dtype=torch.float64)
        for b, L in enumerate(st["kv_lens"]):
            w = st["weights"][b, :L].tolist()
            last = max(case["sinks"], L - case["recent"])
            middle = sorted(range(case["sinks"], last), key=lambda i: (-w[i], i)) if L > case["keep"] else []
            middle = middle[:case["keep"] - case["sinks"] - case["recent"]]
            stay = sorted([*range(case["sinks"]), *middle, *range(last, L)]) if L > case["keep"] else range(L)
            kept[b, :min(L, case["keep"])] = torch.tensor([w[i] for i in stay], dtype=torch.float64)
        return None, None, kept
    if op == "move":
        st = prepare(case, seed)
        held = [t.to(torch.float64) for t in (st["latent"], st["rope"], st["scale"]) if t is not None]
        page, old = case["page"], [t.clone() for t in held]
        for b, (count, first) in enumerate(zip(st["counts"].tolist(), st["first"].tolist())):
            source = st["positions"][b, :count].long()
            target = torch.arange(first, first + count, device=DEV)
            for t, was in zip(held, old):
                t[st["to_table"][b].long()[target // page], target % page] = \
                    was[st["table"][b].long()[source // page], source % page]
        return held
    w = work(case)["flops"]
    st = prepare(case, seed)
    f64 = torch.float64
    new, kv = st["new"], st["kv_lens"]
    pairs = sum(n * L for n, L in zip(new, kv)) * case["H"]
    if w > 1e12 or pairs * (case["N"] if op == "prompt" else case["R"]) > 2e12:
        return None
    total = st["previous"].to(f64) if op == "weights" else None
    outs, lses = [], []
    q_at, k_at = 0, 0
    for b, (n, L) in enumerate(zip(new, kv)):
        # what query i sees of key j, from the definition
        sees = torch.zeros((n, L), dtype=torch.bool, device=DEV)
        j = torch.arange(L, device=DEV)
        if op == "tree":
            sees[:, :L - n] = True
            parent = st["parents"][q_at:q_at + n].tolist()
            pairs = []
            for i in range(n):
                node = i
                while node >= 0:
                    pairs.append((i, L - n + node))
                    node = parent[node]
            both = torch.tensor(pairs, device=DEV)
            sees[both[:, 0], both[:, 1]] = True
        else:
            where = L - n + torch.arange(n, device=DEV)[:, None]
            sees = j.expand(n, L) <= where
            if op != "weights":
                sees = sees & ((where - j < case["window"]) | (j < case["sinks"]))
        if op == "prompt":
            rows = st["kv"][k_at:k_at + L].to(f64)
        else:
            page, use = case["page"], (L + case["page"] - 1) // case["page"]
            ids = st["table"][b, :use].long()
            parts = [st["latent"][ids].reshape(use * page, case["R"])[:L].to(f64)]
            if st["rope"] is not None:
                parts.append(st["rope"][ids].reshape(use * page, case["P"])[:L].to(f64))
            rows = torch.cat(parts, 1)
            if st["scale"] is not None:
                rows = rows * st["scale"][ids].reshape(use * page)[:L, None].to(f64)
        per_o, per_l = [], []
        for h in range(case["H"]):
            if op == "prompt":
                q = st["q"][q_at:q_at + n, h].to(f64)
                keys, values = rows[:, h, :case["N"]], rows[:, h, case["N"]:].contiguous()
                if case["P"]:
                    keys = torch.cat([keys, st["k_rope"][k_at:k_at + L].to(f64)], 1)
            else:
                q = st["q_latent"][q_at:q_at + n, h].to(f64)
                if st["q_rope"] is not None:
                    q = torch.cat([q, st["q_rope"][q_at:q_at + n, h].to(f64)], 1)
                keys, values = rows, rows[:, :case["R"]]
            s = torch.where(sees, q @ keys.T.contiguous() * st["sm"], -math.inf)
            if op == "weights":
                mine = st["lse"][q_at:q_at + n, h, None].to(f64)
                total[b, :L] += torch.where(sees, (s - mine).exp(), 0.0).sum(0)
                continue
            z = torch.logsumexp(s, 1)
            p = torch.where(sees, (s - torch.where(z == -math.inf, 0.0, z)[:, None]).exp(), 0.0)
            per_o.append(p @ values)
            per_l.append(z)
        if op != "weights":
            outs.append(torch.stack(per_o, 1))
            lses.append(torch.stack(per_l, 1))
        q_at, k_at = q_at + n, k_at + L
    if op == "weights":
        return total
    got = (torch.cat(outs), torch.cat(lses)) if case["lse"] else (torch.cat(outs),)
    if op == "tree":
        return (*got, None, None)
    return got if case["lse"] else got[0]
