"""GPU attention over parts of a latent context (windows with first tokens, trees of drafts, the weights each token
receives) against the formulas in 64 bits; tests/context_reference.py states the bounds."""

from __future__ import annotations

import math
import random

import pytest
import torch

from tests import context_reference as cref
from tests import latent_reference as ref
from tests.test_gpu_latent_attention import BF16, DIMS, E4M3, HEADS, _bounds, _expanded_inputs, _i32, _la, _Paged, _queries, _randn

pytestmark = pytest.mark.gpu


def _lc():
    from fused_cpp_amd import latent_context

    return latent_context


def _starts(new):
    return [sum(new[:b]) for b in range(len(new) + 1)]


# ---- windows, absorbed ---------------------------------------------------------------------------------------------


def _forget(pg, lens, keeps):
    """What no query sees is gone: its rows NaN, and the table entries of pages without a seen row no page ids."""
    page = pg.cache.latent.shape[1]
    table = pg.table.cpu()
    for b, keep in enumerate(keeps):
        seen = keep.any(0).cpu()
        for j in range(lens[b]):
            if not seen[j]:
                i = int(table[b, j // page])
                for t in (pg.cache.latent, pg.cache.rope):
                    if t is not None:
                        t.view(torch.uint8)[i, j % page] = 0xff  # NaN in both types
                if pg.cache.scale is not None:
                    pg.cache.scale[i, j % page] = math.nan
        for i in range((lens[b] + page - 1) // page):
            if not bool(seen[i * page:min((i + 1) * page, lens[b])].any()):
                table[b, i] = -1 if i % 2 else 2 ** 31 - 1
    pg.table = table.cuda()


def _check_window(pg, lens, ql, qr, new, scale, window, sinks, starts=True, forget=False, **kw):
    keeps = [cref.seen_by_window(n, L, window, sinks) for n, L in zip(new, lens)]
    st = _starts(new)
    want, wl, tol, ltol = cref.absorbed(ql, qr, pg.rows, st, scale, keeps)
    if forget:
        _forget(pg, lens, keeps)
    out, lse = _la().absorbed_attention(ql, qr, pg.cache, pg.table, pg.lens, scale=scale, window=window, sinks=sinks,
                                        query_starts=_i32(st) if starts else None, return_lse=True, **kw)
    ref.assert_within(out, want, tol, "out")
    ref.assert_within(lse, wl, ltol, "lse")
    return out, lse


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("R,P", DIMS)
@pytest.mark.parametrize("H,n", [(1, 1), (16, 1), (5, 5), (64, 1), (128, 1), (33, 4)])
def test_window_matches(gpu, H, n, R, P, dtype):
    """Every kernel form, lengths around tiles and windows, the rest of the context gone."""
    lens = [0, 1, 2, 63, 64, 65, 130, 200, 777]
    for window, sinks in ((1, 0), (64, 4), (65, 0), (100, 130), (190, 1)):
        pg = _Paged(H + n, lens, R, P, dtype, page=16)
        ql, qr = _queries(H, len(lens) * n, H, R, P)
        _check_window(pg, lens, ql, qr, [n] * len(lens), 0.07, window, sinks, forget=True)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("page", [1, 7, 48, 64, 100, 1000])
def test_window_pages(gpu, page, dtype):
    lens = [1, 130, 2000, 64, 333]
    for window, sinks in ((70, 3), (500, 65)):
        pg = _Paged(page, lens, 512, 64, dtype, page=page, joint=True)
        ql, qr = _queries(2, 5, 16, 512, 64)
        _check_window(pg, lens, ql, qr, [1] * 5, 0.07, window, sinks, starts=False, forget=True)


@pytest.mark.parametrize("H", [1, 16, 128])
@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_window_ragged_queries(gpu, H, dtype):
    """Sequences of no, one and many query tokens, more than keys, chunks longer than the window."""
    new, lens = [0, 1, 40, 3, 7, 0, 2, 150], [50, 0, 20, 900, 7, 0, 1, 700]
    for window, sinks in ((33, 2), (1, 70), (100000, 5)):
        pg = _Paged(H, lens, 512, 64, dtype, page=32)
        ql, qr = _queries(3, sum(new), H, 512, 64)
        out, lse = _check_window(pg, lens, ql, qr, new, 0.07, window, sinks, forget=True)
        assert torch.equal(out[0], torch.zeros_like(out[0])) and bool((lse[0] == -math.inf).all())


@pytest.mark.parametrize("H", [16, 64, 128])
@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_window_long(gpu, H, dtype):
    """A window shared by many workgroups behind a long context; repeated calls give the same bits."""
    lens = [40000, 3, 9000]
    pg = _Paged(7, lens, 512, 64, dtype, page=64)
    ql, qr = _queries(4, 3, H, 512, 64)
    out, lse = _check_window(pg, lens, ql, qr, [1] * 3, 0.07, 4096, 4, starts=False)
    again = _la().absorbed_attention(ql, qr, pg.cache, pg.table, pg.lens, scale=0.07, window=4096, sinks=4, return_lse=True)
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_window_many_sequences(gpu, dtype):
    """More sequences than a wave has lanes and than there are shares, windows of several tiles and of none."""
    count = 300
    lens = [(37 * b) % 450 if b % 5 else 0 for b in range(count)]
    lens[3], lens[count - 1] = 6000, 1
    pg = _Paged(5, lens, 256, 64, dtype, page=32)
    ql, qr = _queries(6, count, 33, 256, 64)
    for window, sinks in ((40, 3), (300, 0)):
        _check_window(pg, lens, ql, qr, [1] * count, 0.07, window, sinks, starts=False)


def test_window_wider_than_the_context_is_none(gpu):
    """The same bits as without a window."""
    la = _la()
    lens = [700, 64, 0, 3000]
    for H, n in ((16, 1), (128, 2)):
        pg = _Paged(9, lens, 512, 64, BF16, page=64)
        ql, qr = _queries(7, 4 * n, H, 512, 64)
        st = _i32([n * b for b in range(5)])
        want = la.absorbed_attention(ql, qr, pg.cache, pg.table, pg.lens, scale=0.07, query_starts=st, return_lse=True)
        for window, sinks in ((3000, 0), (2 ** 40, 2 ** 35), (5000, 17)):
            got = la.absorbed_attention(ql, qr, pg.cache, pg.table, pg.lens, scale=0.07, query_starts=st, window=window,
                                        sinks=sinks, return_lse=True)
            bound = 4 * ref.U * (want[0].abs().to(ref.F64) + 1)
            ref.assert_within(got[0], want[0].to(ref.F64), bound)  # other splits: two results within their bounds


@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_window_growing_scores(gpu, dtype):
    """Scores that rise and fall by far more than the reference point's slack within and between windows."""
    lens, H = [900, 500], 16
    pg = _Paged(11, lens, 512, 64, dtype, page=16)
    ql, qr = _queries(8, 6, H, 512, 64, std=12.0)
    _check_window(pg, lens, ql, qr, [3, 3], 0.07, 200, 66)


def test_window_strides_outputs_and_uncovered(gpu):
    la = _la()
    lens, new, H = [300, 200], [2, 3], 16
    pg = _Paged(13, lens, 512, 64, BF16, page=16)
    wide = _randn(14, 9, H + 3, 640).to(BF16)
    ql, qr = wide[2:7, 1:H + 1, 8:520], wide[2:7, 1:H + 1, 520:584]
    _check_window(pg, lens, ql, qr, new, 0.07, 100, 5)
    # Nine tokens to two sequences may go to another row group than five, whose sums are in another order: each is off
    # the exact value by at most its bound.
    want, _, tol, _ = cref.absorbed(ql, qr, pg.rows, _starts(new), 0.07,
                                    [cref.seen_by_window(n, L, 100, 5) for n, L in zip(new, lens)])
    table = torch.zeros((2, 2 * pg.table.shape[1]), dtype=torch.int32, device="cuda")
    table[:, ::2] = pg.table
    st = _i32([2, 4, 7])
    qs = wide[:9, 1:H + 1]
    out = torch.full((9, H, 520), 3.0, dtype=BF16, device="cuda")
    got, lse = la.absorbed_attention(qs[..., 8:520], qs[..., 520:584], pg.cache, table[:, ::2], pg.lens, scale=0.07, window=100,
                                     sinks=5, query_starts=st, out=out[..., 4:516], return_lse=True)
    ref.assert_within(got[2:7], want, tol)
    assert bool((out[:2] == 3).all()) and bool((out[7:] == 3).all())
    assert bool((out[..., :4] == 3).all()) and bool((out[..., 516:] == 3).all())
    assert bool((lse[:2] == -math.inf).all()) and bool((lse[7:] == -math.inf).all())
    got = la.absorbed_attention(qs[..., 8:520], qs[..., 520:584], pg.cache, table[:, ::2], pg.lens, scale=0.07, window=100,
                                sinks=5, query_starts=st)
    ref.assert_within(got[2:7], want, tol)
    assert bool((got[:2] == 0).all()) and bool((got[7:] == 0).all())


@pytest.mark.parametrize("H", [16, 128])
def test_window_bad_page_within_reach(gpu, H):
    """A page id outside the cache that the window reaches makes the sequence NaN, and no other."""
    lens = [300, 300, 300]
    pg = _Paged(15, lens, 512, 64, BF16, page=16)
    ql, qr = _queries(9, 3, H, 512, 64)
    want = _la().absorbed_attention(ql, qr, pg.cache, pg.table, pg.lens, scale=0.07, window=50, sinks=2)
    pg.table[1, 16] = 10 ** 6  # positions 256 .. 271
    got = _la().absorbed_attention(ql, qr, pg.cache, pg.table, pg.lens, scale=0.07, window=50, sinks=2)
    assert torch.isnan(got[1]).all() and torch.equal(got[0::2], want[0::2])


# ---- windows, expanded ---------------------------------------------------------------------------------------------


def _check_prompt(q, kv, kr, new, lens, scale, window, sinks, **kw):
    qs, ks = _starts(new), _starts(lens)
    keeps = [cref.seen_by_window(n, L, window, sinks) for n, L in zip(new, lens)]
    out, lse = _la().expanded_attention(q, kv, kr, _i32(qs), kv_starts=_i32(ks), scale=scale, window=window, sinks=sinks,
                                        return_lse=True, **kw)
    want, wl, tol, ltol = cref.expanded(q, kv, kr, qs, ks, scale, keeps)
    ref.assert_within(out, want, tol, "out")
    ref.assert_within(lse, wl, ltol, "lse")
    return out, lse


@pytest.mark.parametrize("N,P", HEADS)
@pytest.mark.parametrize("H", [1, 3])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (64, 4), (100, 0), (129, 65), (500, 130), (10 ** 12, 0)])
def test_prompt_window_matches(gpu, H, N, P, window, sinks):
    new, lens = [1, 63, 0, 64, 65, 200, 40, 128], [1, 63, 50, 100, 900, 200, 20, 129]
    _check_prompt(*_expanded_inputs(H + N, new, lens, H, N, P), new, lens, 0.08, window, sinks)


@pytest.mark.parametrize("new,lens", [([1], [20000]), ([3, 150], [9000, 12000]), ([1, 1, 1], [5000, 1, 0])])
@pytest.mark.parametrize("window,sinks", [(4000, 4), (700, 200)])
def test_prompt_window_split(gpu, new, lens, window, sinks):
    """Few rows: the window's tiles shared by several workgroups."""
    _check_prompt(*_expanded_inputs(3, new, lens, 2, 128, 64), new, lens, 0.08, window, sinks)


@pytest.mark.parametrize("N,P", HEADS)
@pytest.mark.parametrize("window,sinks", [(1024, 0), (1030, 3), (2000, 70), (1500, 700)])
def test_prompt_window_long(gpu, N, P, window, sinks):
    """Blocks of 256 rows whose waves' windows begin and end in different tiles."""
    new, lens = [2500, 300], [2600, 2700]
    _check_prompt(*_expanded_inputs(N + P, new, lens, 2, N, P), new, lens, 0.08, window, sinks)


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("window,sinks", [(1024, 0), (1100, 100), (90, 5)])
def test_prompt_window_growing_scores(gpu, sign, window, sinks):
    """Scores that rise (fall) along the keys by far more than the reference point's slack."""
    new = lens = [2300]
    q, kv, kr = _expanded_inputs(5, new, lens, 1, 128, 64)
    ramp = sign * torch.linspace(-20, 20, 2300, device="cuda")[:, None, None]
    q = q.clone()
    q[..., 0] = 8.0
    kv = kv.clone()
    kv[..., :1] = ramp.to(BF16)
    _check_prompt(q, kv, kr, new, lens, 0.08, window, sinks)


def test_prompt_window_more_queries_than_keys(gpu):
    for new, lens in (([2200], [2140]), ([200, 5], [3, 0])):
        out, lse = _check_prompt(*_expanded_inputs(6, new, lens, 2, 128, 64), new, lens, 0.08, 1030, 2)
        assert bool((out[0] == 0).all()) and bool((lse[0] == -math.inf).all())


def test_prompt_window_agrees_with_decode(gpu):
    """The rows of a prompt's last queries are those of the absorbed form over the same keys (values as keys)."""
    la = _la()
    L, H, window, sinks = 600, 4, 150, 6
    q, kv, kr = _expanded_inputs(8, [L], [L], H, 128, 64)
    a = la.expanded_attention(q, kv, kr, _i32([0, L]), scale=0.08, window=window, sinks=sinks)
    b = la.expanded_attention(q[-50:], kv, kr, _i32([0, 50]), kv_starts=_i32([0, L]), scale=0.08, window=window, sinks=sinks)
    keeps = [cref.seen_by_window(50, L, window, sinks)]
    want, _, tol, _ = cref.expanded(q[-50:], kv, kr, [0, 50], [0, L], 0.08, keeps)
    ref.assert_within(a[-50:], want, tol)
    ref.assert_within(b, want, tol)


# ---- trees of drafts -----------------------------------------------------------------------------------------------


def _tree_parents(kind, n, seed):
    rng = random.Random(seed)
    if kind == "chain":
        return list(range(-1, n - 1))
    if kind == "star":
        return [-1] * n
    if kind == "binary":
        return [(i - 1) // 2 if i else -1 for i in range(n)]
    return [rng.randrange(-1, i) if i else -1 for i in range(n)]


def _pack(parents, words):
    masks, depths = [], []
    for line in cref.lines(parents, 64 * words):
        v = [0] * words
        for a in line:
            v[a // 64] |= 1 << (a % 64)
        masks.append([x - (1 << 64) if x >> 63 else x for x in v])
        depths.append(max(len(line) - 1, 0))
    return masks, depths


@pytest.mark.parametrize("nodes", [1, 2, 63, 64, 65, 128, 200, 1024])
def test_draft_tree(gpu, nodes):
    """Masks and depths, bit for bit: chains, stars, odd parents, sequences without nodes and with too many."""
    sizes = [nodes, 0, 1, max(1, nodes // 2), min(nodes + 70, 1100)]
    parents = []
    for k, n in enumerate(sizes):
        p = _tree_parents(("chain", "star", "star", "binary", "random")[k], n, k)
        parents.append(p)
    parents[3][-1] = len(parents[3])       # not below its own number: a root
    parents[4][len(parents[4]) // 2] = -7
    flat = [99, -5] + [v for p in parents for v in p] + [3]  # tokens of no sequence around them
    starts = [2 + s for s in _starts(sizes)]
    tree = _lc().draft_tree(_i32(flat), _i32(starts), nodes)
    words = (nodes + 63) // 64
    masks, depths = [[0] * words] * 2, [0, 0]
    for p in parents:
        m, d = _pack(p, words)
        masks += m
        depths += d
    masks.append([0] * words)
    depths.append(0)
    assert tree.masks.tolist() == masks and tree.depths.tolist() == depths
    assert tree.masks.dtype == torch.int64 and tree.depths.dtype == torch.int32


def test_draft_tree_starts_out_of_order(gpu):
    """A start below an earlier one counts as that one, and starts are cut to the tokens."""
    parents = _i32([-1, 0, 1, -1, 0, 1, 2, 0])
    tree = _lc().draft_tree(parents, _i32([0, 3, 1, 5, 100]), 5)
    want = [([-1, 0, 1]), [], [-1, 0], [-1, 2, 0]]  # tokens 0..2, none, 3..4, 5..7
    m, d = [], []
    for p in want:
        a, b = _pack([v if v < i else -1 for i, v in enumerate(p)], 1)
        m += a
        d += b
    # token 5's parent 1 and 6's parent 2 are not below their own numbers 0 and 1
    assert tree.depths.tolist() == d
    assert tree.masks.tolist() == m


def _check_tree(pg, lens, ql, qr, trees, scale, max_nodes, window=None, sinks=0, **kw):
    new = [len(p) for p in trees]
    st = _i32(_starts(new))
    tree = _lc().draft_tree(_i32([v for p in trees for v in p]), st, max_nodes)
    words = (max_nodes + 63) // 64
    keeps = [cref.seen_by_tree(p, L, window, sinks, words) for p, L in zip(trees, lens)]
    want, wl, tol, ltol = cref.absorbed(ql, qr, pg.rows, _starts(new), scale, keeps)
    if window is not None:
        _forget(pg, lens, keeps)
    out, lse = _la().absorbed_attention(ql, qr, pg.cache, pg.table, pg.lens, scale=scale, query_starts=st, tree=tree,
                                        window=window, sinks=sinks, return_lse=True, **kw)
    ref.assert_within(out, want, tol, "out")
    ref.assert_within(lse, wl, ltol, "lse")
    return out, lse


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("R,P", DIMS)
@pytest.mark.parametrize("H", [1, 5, 16, 128])
def test_tree_matches(gpu, H, R, P, dtype):
    """Contexts of none and more tokens, so that nodes begin at any place of a tile and a mask word."""
    kinds = [("random", 9), ("chain", 5), ("star", 7), ("binary", 33), ("random", 1), ("random", 64)]
    context = [0, 1, 30, 63, 64, 333]
    trees = [_tree_parents(k, n, b) for b, (k, n) in enumerate(kinds)]
    lens = [c + len(p) for c, p in zip(context, trees)]
    pg = _Paged(H, lens, R, P, dtype, page=16)
    ql, qr = _queries(H, sum(map(len, trees)), H, R, P)
    _check_tree(pg, lens, ql, qr, trees, 0.07, 64)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("H", [3, 32])
def test_tree_of_many_nodes(gpu, H, dtype):
    """Masks of several words, nodes over several tiles, at every remainder of the context to a word."""
    for seed, (nodes, context) in enumerate([(65, 1), (130, 17), (200, 40), (257, 95), (100, 31)]):
        trees = [_tree_parents("random", nodes, seed), _tree_parents("chain", nodes // 2, seed)]
        lens = [context + nodes, 3 + nodes // 2]
        pg = _Paged(seed, lens, 512, 64, dtype, page=7)
        ql, qr = _queries(seed, sum(map(len, trees)), H, 512, 64)
        _check_tree(pg, lens, ql, qr, trees, 0.07, nodes)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_tree_behind_a_window(gpu, dtype):
    """Nodes see the context as far as their depth's window goes; what none of them sees may be gone."""
    for H, (window, sinks) in ((16, (70, 3)), (128, (200, 70)), (2, (40, 0))):
        trees = [_tree_parents("random", 12, 1), _tree_parents("chain", 20, 2), _tree_parents("star", 3, 3), [-1]]
        lens = [400 + 12, 30 + 20, 3, 1000]
        pg = _Paged(H, lens, 512, 64, dtype, page=16)
        ql, qr = _queries(H, sum(map(len, trees)), H, 512, 64)
        _check_tree(pg, lens, ql, qr, trees, 0.07, 20, window=window, sinks=sinks)


def test_tree_longer_than_its_sequence(gpu):
    """More nodes than cached tokens: the first nodes have no rows, and nodes past the masks see the context alone."""
    trees = [_tree_parents("chain", 10, 1), _tree_parents("random", 90, 2), _tree_parents("star", 4, 2)]
    lens = [4, 90 + 33, 0]
    pg = _Paged(3, lens, 512, 64, BF16, page=16)
    ql, qr = _queries(3, sum(map(len, trees)), 16, 512, 64)
    out, lse = _check_tree(pg, lens, ql, qr, trees, 0.07, 60)
    assert bool((lse[:6] == -math.inf).all()) and bool((lse[-4:] == -math.inf).all())


def test_tree_of_a_chain_is_causal(gpu):
    """A chain of drafts sees what causal query tokens see."""
    n, H = 7, 16
    lens = [500, 70, 7]
    pg = _Paged(21, lens, 512, 64, BF16, page=16)
    ql, qr = _queries(5, 3 * n, H, 512, 64)
    a, la_ = _check_tree(pg, lens, ql, qr, [_tree_parents("chain", n, 0)] * 3, 0.07, n)
    want, wl, tol, ltol = ref.absorbed(ql, qr, pg.rows, lens, [0, 7, 14, 21], 0.07)
    ref.assert_within(a, want, tol)
    ref.assert_within(la_, wl, ltol)


def test_tree_given_as_masks(gpu):
    """Masks of a user's own: bits beyond a sequence's nodes and rows without any are nothing."""
    lc = _lc()
    L, n, H = 100, 6, 16
    pg = _Paged(22, [L], 512, 64, BF16, page=16)
    ql, qr = _queries(6, n, H, 512, 64)
    bits = [0b000001, 0, 0b111111, ~0, 0b101000, 1 << 40]
    masks = torch.tensor([[b] for b in bits], dtype=torch.int64, device="cuda")
    wide = torch.zeros((n, 3), dtype=torch.int64, device="cuda")
    wide[:, 1:2] = masks
    keep = torch.zeros((n, L), dtype=torch.bool, device="cuda")
    keep[:, :L - n] = True
    for i, b in enumerate(bits):
        for j in range(n):
            keep[i, L - n + j] = bool(b >> j & 1)
    want, wl, tol, ltol = cref.absorbed(ql, qr, pg.rows, [0, n], 0.07, [keep])
    for m in (masks, wide[:, 1:2]):
        out, lse = _la().absorbed_attention(ql, qr, pg.cache, pg.table, pg.lens, scale=0.07, query_starts=_i32([0, n]),
                                            tree=lc.DraftTree(m, torch.zeros(n, dtype=torch.int32, device="cuda")), return_lse=True)
        ref.assert_within(out, want, tol)
        ref.assert_within(lse, wl, ltol)


@pytest.mark.parametrize("H", [16, 128])
def test_tree_long_context(gpu, H):
    trees = [_tree_parents("random", 60, 4), _tree_parents("binary", 9, 4)]
    lens = [20000, 70]
    pg = _Paged(23, lens, 512, 64, BF16, page=64)
    ql, qr = _queries(7, 69, H, 512, 64)
    _check_tree(pg, lens, ql, qr, trees, 0.07, 60)


# ---- the weights each token receives ---------------------------------------------------------------------------------


def _check_weights(pg, lens, ql, qr, new, scale, positions=None, previous=None, starts=True, lse=None, **kw):
    la, lc = _la(), _lc()
    st = _starts(new)
    given = _i32(st) if starts else None
    if lse is None:
        _, lse = la.absorbed_attention(ql, qr, pg.cache, pg.table, pg.lens, scale=scale, query_starts=given, return_lse=True)
    got = lc.attention_weights(ql, qr, pg.cache, pg.table, pg.lens, lse, scale=scale, query_starts=given, previous=previous, **kw)
    S = pg.table.shape[1] * pg.cache.latent.shape[1] if previous is None and positions is None else \
        previous.shape[1] if previous is not None else positions
    want, tol = cref.weights(ql, qr, pg.rows, lens, st, lse, scale, S, previous)
    ref.assert_within(got, want, tol)
    return got, lse


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("R,P", DIMS)
@pytest.mark.parametrize("H,n", [(1, 1), (16, 1), (32, 1), (33, 1), (5, 5), (128, 1), (33, 4), (64, 10)])
def test_weights_match(gpu, H, n, R, P, dtype):
    """Few rows and many, row chunks that do and do not stay in LDS, lengths around the blocks."""
    lens = [0, 1, 2, 63, 127, 128, 129, 255, 257, 777]
    pg = _Paged(H + n, lens, R, P, dtype, page=16)
    ql, qr = _queries(H, len(lens) * n, H, R, P)
    got, lse = _check_weights(pg, lens, ql, qr, [n] * len(lens), 0.07)
    # all of a row's weights are 1: the sums are the rows that see something
    seen = torch.tensor([sum(1 for i in range(n) if L - n + i >= 0) * H for L in lens], device="cuda", dtype=torch.float64)
    assert bool(((got.double().sum(1) - seen).abs() <= 1e-4 * (seen + 1)).all())


@pytest.mark.parametrize("page", [1, 7, 48, 1000])
@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_weights_pages_and_previous(gpu, page, dtype):
    lens = [1, 130, 2000, 0, 333]
    pg = _Paged(page, lens, 512, 64, dtype, page=page, joint=True)
    ql, qr = _queries(2, 5, 16, 512, 64)
    for S in (1, 100, 2500):  # fewer columns than tokens, and more
        previous = torch.rand((5, S), device="cuda") * 3
        _check_weights(pg, lens, ql, qr, [1] * 5, 0.07, previous=previous, starts=False)


@pytest.mark.parametrize("H", [2, 16, 128])
def test_weights_ragged_queries(gpu, H):
    new, lens = [0, 1, 40, 3, 7, 0, 2, 90], [50, 0, 20, 900, 7, 0, 1, 700]
    pg = _Paged(H, lens, 512, 64, BF16, page=32)
    ql, qr = _queries(3, sum(new), H, 512, 64)
    got, _ = _check_weights(pg, lens, ql, qr, new, 0.07)
    assert bool((got[0] == 0).all())
    previous = torch.rand((8, 800), device="cuda")
    got, _ = _check_weights(pg, lens, ql, qr, new, 0.07, previous=previous)
    assert torch.equal(got[0], previous[0]) and torch.equal(got[1], previous[1])


@pytest.mark.parametrize("H,n", [(16, 1), (128, 1), (128, 32)])
def test_weights_in_place_and_repeated(gpu, H, n):
    """out may be previous itself, or the rows of a wider tensor; calls give the same bits."""
    lc = _lc()
    lens = [5000, 3, 900]
    pg = _Paged(31, lens, 512, 64, BF16, page=64)
    ql, qr = _queries(9, 3 * n, H, 512, 64)
    previous = torch.rand((3, 5100), device="cuda")
    st = _i32([n * b for b in range(4)])
    want, lse = _check_weights(pg, lens, ql, qr, [n] * 3, 0.07, previous=previous)
    mine = previous.clone()
    got = lc.attention_weights(ql, qr, pg.cache, pg.table, pg.lens, lse, scale=0.07, query_starts=st, previous=mine, out=mine)
    assert got.data_ptr() == mine.data_ptr() and torch.equal(mine, want)
    wide = torch.full((3, 5200), 7.0, device="cuda")
    wide[:, 50:5150] = previous
    lc.attention_weights(ql, qr, pg.cache, pg.table, pg.lens, lse, scale=0.07, query_starts=st, previous=wide[:, 50:5150],
                         out=wide[:, 50:5150])
    assert torch.equal(wide[:, 50:5150], want) and bool((wide[:, :50] == 7).all()) and bool((wide[:, 5150:] == 7).all())
    spread = torch.rand((5100, 3), device="cuda")
    spread.copy_(previous.T)
    assert torch.equal(lc.attention_weights(ql, qr, pg.cache, pg.table, pg.lens, lse, scale=0.07, query_starts=st,
                                            previous=spread.T), want)


def test_weights_rows_without_a_sum_and_bad_pages(gpu):
    lens, H = [300, 300, 40], 16
    pg = _Paged(32, lens, 512, 64, BF16, page=16)
    ql, qr = _queries(10, 3, H, 512, 64)
    _, lse = _la().absorbed_attention(ql, qr, pg.cache, pg.table, pg.lens, scale=0.07, return_lse=True)
    lse[2] = -math.inf
    lse[1, ::2] = -math.inf
    got, _ = _check_weights(pg, lens, ql, qr, [1] * 3, 0.07, starts=False, lse=lse)
    assert bool((got[2] == 0).all())
    pg.table[1, 3] = -5
    bad = _lc().attention_weights(ql, qr, pg.cache, pg.table, pg.lens, lse, scale=0.07)
    assert torch.isnan(bad[1, 48:64]).all()
    bad[1, 48:64] = got[1, 48:64]
    assert torch.equal(bad, got)


def test_weights_masked_places_may_hold_anything(gpu):
    """NaN in rows that no query of the sequence sees, and in rows that only later queries see."""
    n, H, L = 4, 16, 70
    pg = _Paged(33, [L], 512, 64, BF16, page=16)
    ql, qr = _queries(11, n, H, 512, 64)
    _, lse = _la().absorbed_attention(ql, qr, pg.cache, pg.table, pg.lens, scale=0.07, query_starts=_i32([0, n]), return_lse=True)
    want = _lc().attention_weights(ql, qr, pg.cache, pg.table, pg.lens, lse, scale=0.07, query_starts=_i32([0, n]))
    i, j = int(pg.table[0, (L - 1) // 16]), (L - 1) % 16
    pg.cache.latent[i, j] = math.nan  # only the last query sees it
    got = _lc().attention_weights(ql, qr, pg.cache, pg.table, pg.lens, lse, scale=0.07, query_starts=_i32([0, n]))
    assert torch.isnan(got[0, L - 1]) and torch.equal(got[0, :L - 1], want[0, :L - 1])


# ---- row groups of 128 -------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("R,P", DIMS)
def test_tall_groups_divided_evenly_and_by_parts(gpu, R, P, dtype):
    """Alike groups (cut into equal parts, or whole), one long among short ones (divided evenly), more than there are
    shares; heads that leave waves of the last group without rows."""
    for lens, H, window in (([5000] * 3, 128, 4500), ([900] * 40, 65, 10000), ([3000] + [70] * 30, 97, 10000), ([130] * 300, 128, 40),
                            ([20000], 260, 20000)):
        pg = _Paged(len(lens) + H, lens, R, P, dtype, page=64)
        ql, qr = _queries(H, len(lens), H, R, P)
        out, lse = _check_window(pg, lens, ql, qr, [1] * len(lens), 0.07, window, 3, starts=False)
        again = _la().absorbed_attention(ql, qr, pg.cache, pg.table, pg.lens, scale=0.07, window=window, sinks=3, return_lse=True)
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("sign", [1, -1])
def test_tall_scores_that_grow_and_fall(gpu, dtype, sign):
    """Scores that grow from key to key, so that reference points follow in both halves of a tile, or fall; rows that
    first see a key in a later tile."""
    L, H, R, P = 900, 128, 512, 64
    pg = _Paged(31, [L], R, P, dtype, page=16)
    ramp = sign * torch.linspace(-4, 4, L, device="cuda")
    at = torch.arange(L, device="cuda")
    where = (pg.table[0].long()[at // 16], at % 16)
    if dtype == BF16:
        rows = (pg.rows[0][:, :R] * 0.1 + ramp[:, None]).to(BF16)
        pg.cache.latent[where] = rows
        pg.rows[0][:, :R] = rows.to(ref.F64)
    else:
        before, scale = pg.cache.scale[where].to(ref.F64), (ramp + 4.01) / 100
        pg.cache.scale[where] = scale
        pg.rows[0] = pg.rows[0] / before[:, None] * scale.to(ref.F64)[:, None]  # the first is exact
    ql, qr = _queries(8, 3, H, R, P)
    ql = (ql.float().abs() * 0.3).to(BF16)
    for window, sinks in ((1000, 0), (70, 5), (1, 0)):
        keeps = [cref.seen_by_window(3, L, window, sinks)]
        want, wl, tol, ltol = cref.absorbed(ql, qr, pg.rows, [0, 3], 0.05, keeps)
        out, lse = _la().absorbed_attention(ql, qr, pg.cache, pg.table, pg.lens, scale=0.05, window=window, sinks=sinks,
                                            query_starts=_i32([0, 3]), return_lse=True)
        ref.assert_within(out, want, tol)
        ref.assert_within(lse, wl, ltol)


def test_tall_zero_scales_and_rows_behind(gpu):
    """8-bit rows with a scale of 0 weigh as zeros, in masked tiles too; tokens behind the length may hold anything."""
    L, H = 200, 128
    for window, sinks in ((1000, 0), (100, 3), (7, 0)):
        pg = _Paged(33, [L], 512, 64, E4M3, page=64)
        table = pg.table[0].long()
        at = torch.arange(0, L, 3, device="cuda")
        pg.cache.scale[table[at // 64], at % 64] = 0.0
        pg.rows[0][at] = 0
        ql, qr = _queries(9, 2, H, 512, 64)
        _check_window(pg, [L], ql, qr, [2], 0.07, window, sinks)
