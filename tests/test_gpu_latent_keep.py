"""GPU selection of the positions that stay and moves of cached rows, bit for bit; the operators of a cut-down context
run together, captured, and on streams of their own."""

from __future__ import annotations

import math
import random

import pytest
import torch

from tests import context_reference as cref
from tests.test_gpu_latent_attention import BF16, DIMS, E4M3, _i32, _la, _Paged, _queries, _randn
from tests.test_gpu_latent_context import _lc, _starts, _tree_parents

pytestmark = pytest.mark.gpu


def _check_heaviest(w, lens, keep, sinks, recent):
    positions, counts, kept = _lc().heaviest_positions(w, _i32(lens), keep, sinks=sinks, recent=recent)
    rows = w.cpu().tolist()
    assert positions.dtype == counts.dtype == torch.int32 and positions.shape == kept.shape == (len(lens), keep)
    for b, L in enumerate(lens):
        want = cref.heaviest(rows[b], L, keep, sinks, recent)
        assert int(counts[b]) == len(want), (b, L)
        assert positions[b].tolist() == want + [-1] * (keep - len(want)), (b, L)
        got = kept[b].cpu()
        assert torch.equal(got[:len(want)].nan_to_num(nan=7.5), w[b].cpu()[want].nan_to_num(nan=7.5))
        assert bool((got[len(want):] == 0).all())


@pytest.mark.parametrize("S", [1, 63, 64, 65, 1000, 5000, 8192, 8193, 40000])
@pytest.mark.parametrize("kind", ["heavy", "ties", "zeros", "signs"])
def test_heaviest_matches(gpu, S, kind):
    """Weights as they build up, with many ties, all alike, of both signs with both zeros; counts from 1 to all."""
    g = torch.Generator(device="cuda").manual_seed(S)
    w = torch.randn((4, S), generator=g, device="cuda")
    w = {"heavy": lambda: (2 * w).exp(), "ties": lambda: (w * 2).round(), "zeros": lambda: w * 0,
         "signs": lambda: w * (w.abs() > 0.5)}[kind]()
    if kind == "signs":
        w[:, ::3] = -0.0
    lens = [S, max(0, S - 1), S // 2, 0]
    for keep, sinks, recent in ((1, 0, 0), (max(1, S // 3), 0, 0), (max(1, S // 3), min(4, S // 3), 0), (5, 2, 3), (5, 0, 5),
                                (max(1, S - 1), 1 if S > 1 else 0, 0), (S + 7, 3, 2), (max(8, S // 2), 3, 4)):
        _check_heaviest(w, lens, keep, sinks, recent)


def test_heaviest_infinities_and_nan(gpu):
    w = torch.rand((1, 300), device="cuda")
    w[0, 50], w[0, 60], w[0, 70] = math.inf, -math.inf, math.nan
    w[0, 71] = -torch.tensor(math.nan, device="cuda")
    w[0, 299], w[0, 0] = -math.inf, 1e-45
    for keep in (1, 2, 3, 4, 150, 298, 299):
        _check_heaviest(w, [300], keep, 0, 0)


def test_heaviest_lengths_and_strides(gpu):
    """Lengths past the columns and below 0 are cut; rows of a wider tensor, of a transposed one, the same row for all."""
    wide = torch.rand((3, 700), device="cuda")
    lc = _lc()
    _check_heaviest(wide[:, 100:600], [500, 499, 3], 64, 4, 8)
    a = lc.heaviest_positions(wide[:, 100:600], _i32([10 ** 6, -3, 500]), 64)
    b = lc.heaviest_positions(wide[:, 100:600].contiguous(), _i32([500, 0, 500]), 64)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    _check_heaviest(torch.rand((500, 3), device="cuda").T, [500, 400, 300], 100, 1, 1)
    _check_heaviest(torch.rand((1, 500), device="cuda").expand(3, 500), [500, 400, 99], 100, 1, 1)
    e = lc.heaviest_positions(torch.zeros((0, 5), device="cuda"), _i32([]), 3)
    assert e[0].shape == (0, 3)
    z = lc.heaviest_positions(torch.zeros((2, 0), device="cuda"), _i32([4, 0]), 3)
    assert z[0].tolist() == [[-1] * 3] * 2 and z[1].tolist() == [0, 0] and z[2].tolist() == [[0.0] * 3] * 2


def test_heaviest_of_many_slices(gpu):
    """Long rows: all weights alike, alike but for a few, in one bin of the first digit, and spread; the slices before the
    last that stays empty of what is kept, or full of it."""
    S = 70000
    g = torch.Generator(device="cuda").manual_seed(3)
    w = torch.rand((5, S), generator=g, device="cuda")
    w[0] = 0.5
    w[1] = 0.0
    w[1, 30000:30100] = torch.rand(100, generator=g, device="cuda")
    w[2] = 1 + w[2] * 1e-3
    w[3, :20000] += 1000
    w[4, -9000:] += 1000
    for lens in ([S] * 5, [S - 1, 50000, 8193, 24577, 66000]):
        for keep, sinks, recent in ((1, 0, 0), (9000, 4, 64), (9000, 8990, 10), (20000, 0, 0), (69999, 1, 1), (69000, 9000, 9000)):
            _check_heaviest(w, lens, keep, sinks, recent)


def test_heaviest_many_sequences(gpu):
    w = torch.rand((300, 600), device="cuda").mul_(8).floor_()
    lens = [(b * 7) % 601 for b in range(300)]
    _check_heaviest(w, lens, 100, 3, 5)


# ---- moves -----------------------------------------------------------------------------------------------------------


def _bytes(c):
    return [t.view(torch.uint8) if t.dtype == E4M3 else t for t in (c.latent, c.rope, c.scale) if t is not None]


def _same(c, tensors):
    return all(torch.equal(a.float().nan_to_num(nan=7.5), b.float().nan_to_num(nan=7.5)) for a, b in zip(_bytes(c), tensors))


def _moved(c, table, to_table, positions, counts, starts):
    """What the cache should hold: every row read before any is written."""
    page, pages = c.latent.shape[1], c.latent.shape[0]
    now = [t.clone() for t in _bytes(c)]
    was = [t.clone() for t in now]

    def at(t, b, p):
        if p < 0 or p // page >= t.shape[1]:
            return None
        i = int(t[b, p // page])
        return (i, p % page) if 0 <= i < pages else None

    table, to = table.cpu(), (table if to_table is None else to_table).cpu()
    for b, n in enumerate(counts):
        for k in range(max(0, min(n, len(positions[b])))):
            s, d = at(table, b, positions[b][k]), at(to, b, starts[b] + k)
            if s is not None and d is not None:
                for x, y in zip(now, was):
                    x[d] = y[s]
    return now


def _check_move(pg, positions, counts, starts=None, to_table=None, table=None):
    table = pg.table if table is None else table
    want = _moved(pg.cache, table, to_table, positions, counts, starts or [0] * len(counts))
    _lc().latent_cache_move(pg.cache, table, _i32(positions), _i32(counts), starts=None if starts is None else _i32(starts),
                            to_table=to_table)
    assert _same(pg.cache, want)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("R,P", DIMS)
@pytest.mark.parametrize("page", [1, 7, 16])
def test_move_within(gpu, R, P, dtype, page):
    """Evictions and accepted drafts in their own pages."""
    lens = [300, 1, 0, 200, 64]
    rng = random.Random(page)
    pg = _Paged(page, lens, R, P, dtype, page=page, joint=page == 7)
    kept = [sorted(rng.sample(range(n), n // 2)) for n in lens]
    m = max(map(len, kept))
    _check_move(pg, [k + [-1] * (m - len(k)) for k in kept], [len(k) for k in kept])
    starts = [290, 0, 0, 180, 0]
    kept = [[290, 292, 299], [], [], [185, 186, 199], [3]]
    _check_move(pg, [k + [-1] * (3 - len(k)) for k in kept], [3, 0, 0, 3, 1], starts)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_move_within_many_rows(gpu, dtype):
    """More rows than a workgroup holds at once, by distances of one and of thousands."""
    lens = [5000, 3500]
    pg = _Paged(3, lens, 512, 64, dtype, page=64)
    _check_move(pg, [list(range(1, 5000)), list(range(1000, 3500)) + [-1] * 2499], [4999, 2500])
    rng = random.Random(1)
    kept = [sorted(rng.sample(range(n), 3000)) for n in lens]
    _check_move(pg, kept, [3000, 3000])


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("R,P", DIMS)
@pytest.mark.parametrize("page", [1, 7, 16])
def test_move_apart(gpu, R, P, dtype, page):
    """To other pages, in any order, a row to several places."""
    lens = [300, 1, 0, 200]
    rng = random.Random(page)
    pg = _Paged(page, lens, R, P, dtype, page=page, joint=page == 7, spare=3 + 300)
    used = set(int(v) for b, n in enumerate(lens) for v in pg.table[b, :(n + page - 1) // page].tolist())
    free = [i for i in range(pg.cache.latent.shape[0]) if i not in used]
    width = (210 + page - 1) // page
    to = _i32([[free[b * 70 + i] if b * 70 + i < len(free) and i < 70 else -1 for i in range(width)] for b in range(4)])
    kept = [[rng.randrange(max(1, n)) for _ in range(190)] for n in lens]
    _check_move(pg, kept, [190, 5, 0, 150], [3, 0, 0, 60], to_table=to)


@pytest.mark.parametrize("apart", [True, False])
def test_move_bad_places(gpu, apart):
    """Positions and pages that name no row, counts out of range: those rows are left out, the others move."""
    lens = [100, 100, 100]
    pg = _Paged(5, lens, 512, 64, BF16, page=16, spare=30)
    used = set(pg.table.flatten().tolist())
    free = [i for i in range(pg.cache.latent.shape[0]) if i not in used]
    to = _i32([free[:7], free[7:14], free[14:21]])
    table = pg.table.clone()
    table[0, 2], table[1, 5] = -1, 10 ** 6
    to[0, 1], to[2, 0] = 2 ** 31 - 1, -4
    positions = [[2, 5, 33, 50, 99, 100, 10 ** 6, 2 ** 31 - 1], [0, 1, 20, 81, 82, 97, 98, 99], [-1, -5, 10, 11, 12, 13, 14, 15]]
    if not apart:
        positions[2] = [1, 2, 10, 11, 12, 13, 14, 15]
    _check_move(pg, positions, [10 ** 6, -3, 6], [0, 0, 0], to_table=to if apart else None, table=table)
    _check_move(pg, positions, [8, 8, 8], [2 ** 31 - 1, -1, 0] if apart else [0, 0, 0], to_table=to if apart else None, table=table)


def test_move_strided_tables_and_empty(gpu):
    lens = [100, 60]
    pg = _Paged(6, lens, 512, 64, BF16, page=16, spare=12)
    used = set(pg.table.flatten().tolist())
    free = [i for i in range(pg.cache.latent.shape[0]) if i not in used]
    table = torch.zeros((2, 14), dtype=torch.int32, device="cuda")
    table[:, ::2] = pg.table
    to = torch.zeros((5, 2), dtype=torch.int32, device="cuda")
    to.T[:2] = _i32([free[:5], free[5:10]])
    _check_move(pg, [[50, 3, 99], [1, 2, 3]], [3, 2], to_table=to.T, table=table[:, ::2])
    before = [t.clone() for t in _bytes(pg.cache)]
    lc = _lc()
    lc.latent_cache_move(pg.cache, pg.table, torch.zeros((2, 0), dtype=torch.int32, device="cuda"), _i32([0, 0]))
    lc.latent_cache_move(pg.cache, pg.table[:0], torch.zeros((0, 3), dtype=torch.int32, device="cuda"), _i32([]))
    lc.latent_cache_move(pg.cache, pg.table[:, :0], _i32([[1], [1]]), _i32([1, 1]))
    lc.latent_cache_move(pg.cache, pg.table, _i32([[1], [1]]), _i32([1, 1]), to_table=to.T[:2, :0])
    assert _same(pg.cache, before)


# ---- together ----------------------------------------------------------------------------------------------------------


def _decode_step(pg, ql, qr, weights, keep, scale=0.07):
    la, lc = _la(), _lc()
    o, lse = la.absorbed_attention(ql, qr, pg.cache, pg.table, pg.lens, scale=scale, return_lse=True)
    lc.attention_weights(ql, qr, pg.cache, pg.table, pg.lens, lse, scale=scale, previous=weights, out=weights)
    positions, counts, kept = lc.heaviest_positions(weights, pg.lens, keep, sinks=2, recent=8)
    lc.latent_cache_move(pg.cache, pg.table, positions, counts)
    return o, lse, positions, counts, kept


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("H", [16, 128])
def test_a_cache_cut_down(gpu, H, dtype):
    """Attention over the kept rows is that over the kept positions of the whole context."""
    lens, keep = [900, 50, 333], 100
    pg = _Paged(41, lens, 512, 64, dtype, page=16)
    ql, qr = _queries(12, 3, H, 512, 64)
    weights = torch.zeros((3, 912), device="cuda")
    o, lse, positions, counts, kept = _decode_step(pg, ql, qr, weights, keep)
    keeps = []
    for b, L in enumerate(lens):
        k = torch.zeros((1, L), dtype=torch.bool, device="cuda")
        k[0, positions[b, :int(counts[b])].long()] = True
        keeps.append(k)
    want, wl, tol, ltol = cref.absorbed(ql, qr, pg.rows, [0, 1, 2, 3], 0.07, keeps)
    out, l2 = _la().absorbed_attention(ql, qr, pg.cache, pg.table, counts, scale=0.07, return_lse=True)
    from tests.latent_reference import assert_within

    assert_within(out, want, tol)
    assert_within(l2, wl, ltol)
    assert bool((kept.sum(1) <= weights.sum(1) + 1e-3).all())


@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_drafts_verified(gpu, dtype):
    """A tree's rows, then its accepted line moved behind the context: the next step reads them as a causal sequence."""
    la, lc = _la(), _lc()
    context, H = [200, 64], 16
    trees = [_tree_parents("random", 20, 3), _tree_parents("binary", 15, 3)]
    lens = [c + len(p) for c, p in zip(context, trees)]
    pg = _Paged(42, lens, 512, 64, dtype, page=16)
    new = [len(p) for p in trees]
    st = _i32(_starts(new))
    ql, qr = _queries(13, sum(new), H, 512, 64)
    tree = lc.draft_tree(_i32([v for p in trees for v in p]), st, 20)
    out = la.absorbed_attention(ql, qr, pg.cache, pg.table, pg.lens, scale=0.07, query_starts=st, tree=tree)
    accepted = [sorted(max(cref.lines(p), key=len)) for p in trees]
    m = max(map(len, accepted))
    lc.latent_cache_move(pg.cache, pg.table, _i32([[c + a for a in line] + [-1] * (m - len(line)) for c, line in zip(context, accepted)]),
                         _i32([len(a) for a in accepted]), starts=_i32(context))
    now = [c + len(a) for c, a in zip(context, accepted)]
    last = [s + a[-1] for s, a in zip(_starts(new), accepted)]
    again = la.absorbed_attention(ql[last], None if qr is None else qr[last], pg.cache, pg.table, _i32(now), scale=0.07)
    rows = [torch.cat([r[:c], r[c:][a]]) for r, c, a in zip(pg.rows, context, accepted)]
    keeps = [torch.ones((1, n), dtype=torch.bool, device="cuda") for n in now]
    want, _, tol, _ = cref.absorbed(ql[last], qr[last], rows, [0, 1, 2], 0.07, keeps)
    from tests.latent_reference import assert_within

    assert_within(again, want, tol)
    assert_within(out[last], want, tol)


def test_window_layer_over_freed_pages(gpu):
    """Decode steps of a windowed cache whose pages come back as the window leaves them."""
    la = _la()
    H, page, window, sinks = 16, 16, 50, 3
    cache = la.allocate_latent_cache(6, page)
    free = list(range(6))
    table = torch.full((1, 20), -1, dtype=torch.int32)
    rows = []
    cos_sin = torch.cat([torch.ones(400, 32), torch.zeros(400, 32)], 1).cuda()
    for t in range(300):
        if t % page == 0:
            table[0, t // page] = free.pop()
        gone = (t - window) // page  # the last page that lies before the window whole
        if gone >= 1 and (gone + 1) * page <= t - window + 1 and table[0, gone] >= 0:
            free.append(int(table[0, gone]))
            table[0, gone] = -1
        kv = _randn(t, 1, 576).to(BF16)
        slot = int(table[0, t // page]) * page + t % page
        row = la.latent_cache_append(kv, _i32([t]), _i32([slot]), cos_sin, cache, return_rows=True)
        rows.append(row[0])
        if t % 37 == 0 or t > 290:
            ql, qr = _queries(t, 1, H, 512, 64)
            got = la.absorbed_attention(ql, qr, cache, table.cuda(), _i32([t + 1]), scale=0.07, window=window, sinks=sinks)
            keep = cref.seen_by_window(1, t + 1, window, sinks)
            want, _, tol, _ = cref.absorbed(ql, qr, [torch.stack(rows).double()], [0, 1], 0.07, [keep])
            from tests.latent_reference import assert_within

            assert_within(got, want, tol)


def test_captured(gpu):
    """A tree step and a cut-down step captured once replay with new lengths, parents, weights and pages."""
    la, lc = _la(), _lc()
    H, keep = 16, 40
    lens = [300, 200]
    pg = _Paged(51, lens, 512, 64, BF16, page=16)
    start = [t.clone() for t in (pg.cache.latent, pg.cache.rope)]
    new = [6, 5]
    st = _i32(_starts(new))
    parents = _i32(_tree_parents("random", 6, 1) + _tree_parents("binary", 5, 1))
    ql, qr = _queries(14, 11, H, 512, 64)
    q1, r1 = _queries(15, 2, H, 512, 64)
    weights = torch.zeros((2, 320), device="cuda")

    def step():
        tree = lc.draft_tree(parents, st, 6)
        a = la.absorbed_attention(ql, qr, pg.cache, pg.table, pg.lens, scale=0.07, query_starts=st, tree=tree, window=100, sinks=4)
        b = la.absorbed_attention(ql, qr, pg.cache, pg.table, pg.lens, scale=0.07, query_starts=st, window=60, sinks=2)
        return (a, b, tree.masks, tree.depths, *_decode_step(pg, q1, r1, weights, keep))

    def reset(k):
        pg.cache.latent.copy_(start[0])
        pg.cache.rope.copy_(start[1])
        weights.copy_(torch.rand((2, 320), generator=torch.Generator(device="cuda").manual_seed(k), device="cuda"))
        pg.lens.copy_(_i32([300 - 13 * k, 200 - 50 * k]))
        parents.copy_(_i32(_tree_parents("random", 6, k) + _tree_parents("chain", 5, k)))
        st.copy_(_i32([0, 6, 11] if k % 2 == 0 else [0, 4, 9]))

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        reset(0)
        step()
    stream.synchronize()
    reset(0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in (1, 3, 0, 2, 1):
        reset(k)
        want = [t.clone() for t in step()]
        left = [t.clone() for t in (pg.cache.latent, pg.cache.rope, weights)]
        reset(k)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), k
        assert all(torch.equal(a.nan_to_num(nan=7.5), b.nan_to_num(nan=7.5))
                   for a, b in zip((pg.cache.latent, pg.cache.rope, weights), left)), k


def test_side_streams(gpu):
    """Two calls at once on streams of their own, each with its workspace."""
    la, lc = _la(), _lc()
    H, lens = 128, [6000, 100]
    pg = _Paged(61, lens, 512, 64, BF16, page=64)
    ql, qr = _queries(16, 2 * 16, H, 512, 64)
    st = _i32([0, 16, 32])

    def run():
        o, lse = la.absorbed_attention(ql, qr, pg.cache, pg.table, pg.lens, scale=0.07, query_starts=st, window=3000, sinks=4, return_lse=True)
        return o, lse, lc.attention_weights(ql, qr, pg.cache, pg.table, pg.lens, lse, scale=0.07, query_starts=st)

    want = run()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got[i].append(run())
    torch.cuda.synchronize()
    for r in got[0] + got[1]:
        assert all(torch.equal(a, b) for a, b in zip(r, want))
