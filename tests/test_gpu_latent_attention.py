"""GPU latent attention against the formulas in 64 bits (tests/latent_reference.py states the bounds)."""

from __future__ import annotations

import math

import pytest
import torch

from tests import latent_reference as ref

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
E4M3 = torch.float8_e4m3fn


def _la():
    from fused_cpp_amd import latent_attention

    return latent_attention


def _randn(seed, *shape, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda") * std


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ---- norm and rotation -------------------------------------------------------------------------------------------


def _check_norm_rope(x, pos, table, weight, normalize, inverse, interleaved, eps, **kw):
    got = _la().head_norm_rope(x, pos, table, weight=weight, normalize=normalize, inverse=inverse,
                               interleaved=interleaved, eps=eps, **kw)
    y = x.to(ref.F64)
    if normalize:
        y = ref.norm(y, weight, eps)
    want, mag = ref.rotate(y, table[pos.long()], interleaved, inverse)
    ref.assert_within(got, want, ref.U * want.abs() + (x.shape[-1] + 32) * ref.E * mag + 1e-38)
    return got


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("T,H,D,P", [(1, 1, 64, 64), (3, 128, 192, 64), (17, 5, 128, 0), (9, 64, 512, 64), (33, 3, 576, 64),
                                     (5, 2, 1024, 128), (4, 3, 1032, 16), (7, 3, 70, 30), (2, 4, 9, 2), (6, 2, 40, 24),
                                     (4099, 7, 64, 32)])
def test_norm_rope_matches(gpu, T, H, D, P, interleaved):
    x = _randn(T + D, T, H, D, std=3.0).to(BF16)
    table = ref.rope_table(P, 1000, "cuda")
    pos = torch.randint(0, 1000, (T,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(T))
    w = (1 + 0.2 * _randn(D, D)).to(BF16)
    _check_norm_rope(x, pos, table, w, True, False, interleaved, 1e-6)
    _check_norm_rope(x, pos.int(), table, None, True, True, interleaved, 1e-3)
    _check_norm_rope(x, pos, table, None, False, False, interleaved, 1e-6)


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("D,P", [(192, 64), (70, 30)])
def test_norm_rope_in_place_and_strided(gpu, D, P, interleaved):
    """x itself as the output, views of a wider tensor, transposed heads, values that are not contiguous."""
    la = _la()
    table = ref.rope_table(P, 50, "cuda")
    pos = torch.arange(11, device="cuda")
    wide = _randn(5, 11, 6, D + 24).to(BF16)
    x = wide[:, :, 8:8 + D]
    before = wide.clone()
    want = _check_norm_rope(x, pos, table, None, True, False, interleaved, 1e-6)
    out = la.head_norm_rope(x, pos, table, interleaved=interleaved, out=x)
    assert out.data_ptr() == x.data_ptr()
    assert torch.equal(x, want)
    assert torch.equal(wide[:, :, :8], before[:, :, :8]) and torch.equal(wide[:, :, 8 + D:], before[:, :, 8 + D:])
    odd = _randn(6, 11, 6, D + 3).to(BF16)[:, :, 3:]  # rows at odd multiples of 2 bytes
    _check_norm_rope(odd, pos, table, None, True, False, interleaved, 1e-6)
    _check_norm_rope(_randn(7, 6, 11, D).to(BF16).transpose(0, 1), pos, table, None, True, True, interleaved, 1e-6)
    _check_norm_rope(_randn(8, 11, D, 6).to(BF16).transpose(1, 2), pos, table, None, True, False, interleaved, 1e-6)
    spread = torch.zeros((11, 6, D, 2), dtype=BF16, device="cuda")
    _check_norm_rope(_randn(9, 11, 6, D).to(BF16), pos, table, None, True, False, interleaved, 1e-6,
                     out=spread[..., 0])
    one = _randn(10, 1, 6, D).to(BF16).expand(11, 6, D)  # the same row for every token
    _check_norm_rope(one, pos, table, None, True, False, interleaved, 1e-6)


def test_norm_rope_back_and_zero_rows(gpu):
    la = _la()
    table = ref.rope_table(64, 4096, "cuda")
    x = _randn(1, 64, 8, 192).to(BF16)
    pos = torch.arange(64, device="cuda") * 63
    back = la.head_norm_rope(la.head_norm_rope(x, pos, table, normalize=False), pos, table, normalize=False, inverse=True)
    # two roundings of values at most |a| + |b|
    y, mag = ref.rotate(x.to(ref.F64), table[pos] * 0 + torch.cat([torch.ones(32), torch.zeros(32)]).cuda(), True, False)
    ref.assert_within(back, y, 3 * ref.U * mag)
    z = la.head_norm_rope(torch.zeros((3, 2, 192), dtype=BF16, device="cuda"), pos[:3], table)
    assert torch.equal(z, torch.zeros_like(z))
    assert la.head_norm_rope(x[:0], pos[:0], table).shape == (0, 8, 192)


def test_norm_rope_position_outside_the_table(gpu):
    table = ref.rope_table(64, 10, "cuda")
    x = _randn(2, 4, 3, 192).to(BF16)
    for D in (192, 190):
        y = _la().head_norm_rope(x[:, :, :D], torch.tensor([0, 10, -1, 9], device="cuda"), table, normalize=False)
        assert torch.isnan(y[1:3, :, D - 64:]).all()
        assert torch.equal(y[1:3, :, :D - 64], x[1:3, :, :D - 64])
        assert torch.isfinite(y[0::3]).all()


# ---- the cache ---------------------------------------------------------------------------------------------------


def _cache(pages, page, R, P, dtype, fill=None, joint=False):
    la = _la()
    if joint:  # latent and key part as views of one tensor
        both = torch.zeros((pages, page, R + P), dtype=BF16 if dtype == BF16 else torch.uint8, device="cuda").view(dtype)
        scale = torch.zeros((pages, page), device="cuda") if dtype == E4M3 else None
        c = la.LatentCache(both[..., :R], both[..., R:] if P else None, scale)
    else:
        c = la.allocate_latent_cache(pages, page, latent_dim=R, rope_dim=P, dtype=dtype)
    if fill is not None:
        for t in (c.latent, c.rope):
            if t is not None:
                t.copy_(torch.full(t.shape, fill, device="cuda").to(dtype))
        if c.scale is not None:
            c.scale.fill_(fill)
    return c


def _cache_rows(c, slots):
    """The values of cached rows."""
    page = c.latent.shape[1]
    i, j = slots // page, slots % page
    rows = c.latent[i, j].to(ref.F64)
    if c.rope is not None:
        rows = torch.cat([rows, c.rope[i, j].to(ref.F64)], 1)
    return rows if c.scale is None else rows * c.scale[i, j].to(ref.F64)[:, None]


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("R,P,rot", [(512, 64, 64), (512, 0, 64), (256, 64, 64), (256, 0, 256), (512, 0, 0)])
def test_append_matches(gpu, R, P, rot, dtype, interleaved):
    la = _la()
    T, pages, page = 61, 9, 13
    c = _cache(pages, page, R, P, dtype, joint=rot == 64)
    kv = _randn(R + P, T, R + P, std=2.0).to(BF16)
    kv[5] = 0
    kv[6, :R] *= 1e-3
    slots = torch.randperm(pages * page, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))[:T]
    slots[7], slots[11] = -1, pages * page  # padding, and a slot behind the last page
    pos = torch.arange(T, device="cuda") * 5
    table = ref.rope_table(rot, 400, "cuda")
    w = (1 + 0.2 * _randn(1, R)).to(BF16)
    before = [None if t is None else t.clone() for t in (c.latent, c.rope, c.scale)]
    rows = la.latent_cache_append(kv, pos.int(), slots, table, c, weight=w, interleaved=interleaved, return_rows=True)
    x = kv.to(ref.F64)
    want, mag = ref.rotate(torch.cat([ref.norm(x[:, :R], w, 1e-6), x[:, R:]], 1), table[pos], interleaved, False)
    small = (R + 64) * ref.E * mag
    ref.assert_within(rows, want, ref.U * want.abs() + small)
    kept = torch.tensor([t for t in range(T) if t not in (7, 11)], device="cuda")
    got = _cache_rows(c, slots[kept])
    if dtype == BF16:
        assert torch.equal(got, rows[kept].to(ref.F64))
    else:
        top = want[kept].abs().amax(1, keepdim=True)
        scale = torch.where(top > 0, top / 448, torch.ones_like(top))
        s = c.scale.view(-1)[slots[kept]].to(ref.F64)[:, None]
        ref.assert_within(s, scale, (R + 64) * ref.E * scale)
        ref.assert_within(got, want[kept], 2.0 ** -4 * want[kept].abs() + 2.0 ** -10 * scale + 2 * small[kept] +
                          448 * scale * (R + 64) * ref.E)
    # everything else is as it was
    mine = torch.zeros(pages * page, dtype=torch.bool, device="cuda")
    mine[slots[kept]] = True
    for t, b in zip((c.latent, c.rope, c.scale), before):
        if t is not None:
            a, b = (u.contiguous().view(torch.uint8).reshape(pages * page, -1) for u in (t, b))
            assert torch.equal(a[~mine], b[~mine])
    # without the rows, int32 slots, a strided kv: the same cache
    c2 = _cache(pages, page, R, P, dtype)
    wide = torch.zeros((T, R + P + 5), dtype=BF16, device="cuda")
    wide[:, 5:] = kv
    assert la.latent_cache_append(wide[:, 5:], pos, slots.int(), table, c2, weight=w, interleaved=interleaved) is None
    assert torch.equal(_cache_rows(c2, slots[kept]), got)


def test_append_edges(gpu):
    la = _la()
    table = ref.rope_table(64, 16, "cuda")
    c = _cache(2, 4, 512, 64, E4M3)
    kv = _randn(1, 3, 576).to(BF16)
    pos = torch.tensor([1, 99, 2], device="cuda")
    la.latent_cache_append(kv[:0], pos[:0], pos[:0], table, c)
    la.latent_cache_append(kv, pos, torch.tensor([0, 1, 2], device="cuda"), table, c)
    rows = _cache_rows(c, torch.arange(3, device="cuda"))
    assert torch.isnan(rows[1, 512:]).all() and torch.isfinite(rows[0::2]).all()
    empty = _cache(0, 4, 512, 64, BF16)
    got = la.latent_cache_append(kv, pos, torch.tensor([0, 1, 2], device="cuda"), table, empty, return_rows=True)
    assert got.shape == (3, 576)
    big = kv.clone()
    big[0, 512:] = 1e30  # a row whose key part dwarfs the latent
    la.latent_cache_append(big, torch.zeros_like(pos), torch.tensor([5, 6, 7], device="cuda"), table, c)
    v = _cache_rows(c, torch.tensor([5], device="cuda"))
    assert torch.isfinite(v).all() and float((v[0, 512:] / big[0, 512:].to(ref.F64) - 1).abs().max()) <= 2.0 ** -4


# ---- per-head products -----------------------------------------------------------------------------------------------


@pytest.mark.parametrize("T", [1, 15, 16, 17, 64, 65, 200])
@pytest.mark.parametrize("H,N,K", [(128, 512, 128), (3, 128, 512), (5, 64, 72), (1, 8, 8), (2, 136, 40), (7, 24, 256)])
def test_head_projection_matches(gpu, T, H, N, K):
    la = _la()
    w = _randn(N, H, N, K).to(BF16)
    x = _randn(K, T, H, K + 8).to(BF16)[..., :K]
    got = la.head_projection(x, la.prepare_head_projection(w))
    a, b = x.to(ref.F64).transpose(0, 1).contiguous(), w.to(ref.F64).transpose(1, 2).contiguous()
    want, mag = (a @ b).transpose(0, 1), (a.abs() @ b.abs()).transpose(0, 1)
    ref.assert_within(got, want, ref.U * want.abs() + K * ref.E * mag)


def test_head_projection_layouts(gpu):
    la = _la()
    kv_b = _randn(1, 4, 128 + 128, 512).to(BF16)  # both up-projections of a layer in one weight
    w_uk, w_uv = kv_b[:, :128].transpose(1, 2), kv_b[:, 128:]
    q = _randn(2, 9, 4, 192).to(BF16)
    a = la.head_projection(q[..., :128], la.prepare_head_projection(w_uk))
    assert torch.equal(a, la.head_projection(q[..., :128].contiguous(), la.prepare_head_projection(w_uk.contiguous())))
    out = torch.full((9, 4, 130), 3.0, dtype=BF16, device="cuda")
    p = la.prepare_head_projection(w_uv)
    want = la.head_projection(a, p)
    assert la.head_projection(a, p, out=out[..., 1:129]).data_ptr() == out[..., 1:].data_ptr()
    assert torch.equal(out[..., 1:129], want) and bool((out[..., 0] == 3).all()) and bool((out[..., 129] == 3).all())
    assert torch.equal(la.head_projection(a.transpose(0, 1).contiguous().transpose(0, 1), p), want)
    assert la.head_projection(a[:0], p).shape == (0, 4, 128)


# ---- absorbed attention ------------------------------------------------------------------------------------------------


class _Paged:
    """Sequences' rows scattered over a cache whose other rows are NaN."""

    def __init__(self, seed, lens, R, P, dtype, page, std=1.0, joint=False, spare=3):
        la = _la()
        used = [(n + page - 1) // page for n in lens]
        pages = sum(used) + spare
        self.cache = _cache(pages, page, R, P, dtype, fill=math.nan, joint=joint)
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
        width = max(used + [1])
        table = torch.full((len(lens), width), 2 ** 31 - 1, dtype=torch.int32)  # entries past a length are not ids
        self.rows = []
        for b, n in enumerate(lens):
            ids = [order.pop() for _ in range(used[b])]
            table[b, :used[b]] = torch.tensor(ids, dtype=torch.int32)
            x = _randn(seed * 100 + b, n, R + P, std=std).to(BF16)
            j = torch.arange(n, device="cuda")
            i = torch.tensor(ids or [0], device="cuda")[j // page] if n else j
            if dtype == E4M3:
                s = x.float().abs().amax(1) / 448 if n else x.float()[:, 0]
                x8 = (x.float() / s[:, None]).to(E4M3)
                self.cache.scale[i, j % page] = s
                self.cache.latent.view(torch.uint8)[i, j % page] = x8.view(torch.uint8)[:, :R]
                if P:
                    self.cache.rope.view(torch.uint8)[i, j % page] = x8.view(torch.uint8)[:, R:]
                self.rows.append(x8.to(ref.F64) * s.to(ref.F64)[:, None])
            else:
                self.cache.latent[i, j % page] = x[:, :R]
                if P:
                    self.cache.rope[i, j % page] = x[:, R:]
                self.rows.append(x.to(ref.F64))
        self.table = table.cuda()
        self.lens = _i32(lens)


def _queries(seed, T, H, R, P, std=1.5):
    q = _randn(seed, T, H, R + P, std=std).to(BF16)
    return q[..., :R], (q[..., R:] if P else None)


def _check_absorbed(pg, lens, ql, qr, starts, scale, **kw):
    la = _la()
    st = None if starts is None else _i32(starts)
    out, lse = la.absorbed_attention(ql, qr, pg.cache, pg.table, pg.lens, scale=scale, query_starts=st, return_lse=True, **kw)
    want, wl, tol, ltol = ref.absorbed(ql, qr, pg.rows, lens, starts or list(range(len(lens) + 1)), scale)
    ref.assert_within(out, want, tol, "out")
    ref.assert_within(lse, wl, ltol, "lse")
    return out, lse


DIMS = [(512, 64), (512, 0), (256, 64), (256, 0)]


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("R,P", DIMS)
@pytest.mark.parametrize("H,n", [(1, 1), (16, 1), (16, 2), (5, 5), (64, 1), (128, 1), (33, 4)])
def test_absorbed_matches(gpu, H, n, R, P, dtype):
    """Every kernel form (16, 32, 64, 128 rows), odd heads, several query tokens, lengths around the tile."""
    lens = [0, 1, 2, 63, 64, 65, 128, 200, 777]
    pg = _Paged(H + n, lens, R, P, dtype, page=16)
    ql, qr = _queries(H, len(lens) * n, H, R, P)
    _check_absorbed(pg, lens, ql, qr, [n * b for b in range(len(lens) + 1)], 0.07)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("page", [1, 7, 48, 64, 100, 1000])
def test_absorbed_pages(gpu, page, dtype):
    lens = [1, 130, 500, 64]
    pg = _Paged(page, lens, 512, 64, dtype, page=page, joint=True)
    ql, qr = _queries(2, 4, 16, 512, 64)
    _check_absorbed(pg, lens, ql, qr, None, 0.07)


@pytest.mark.parametrize("H", [16, 128])
@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_absorbed_ragged_queries(gpu, H, dtype):
    """Sequences of no, one and many query tokens; more query tokens than keys leave rows that see nothing."""
    new, lens = [0, 1, 40, 3, 7, 0, 2], [50, 0, 20, 900, 7, 0, 1]
    starts = [sum(new[:b]) for b in range(len(new) + 1)]
    pg = _Paged(H, lens, 512, 64, dtype, page=32)
    ql, qr = _queries(3, sum(new), H, 512, 64)
    out, lse = _check_absorbed(pg, lens, ql, qr, starts, 0.07)
    assert torch.equal(out[0], torch.zeros_like(out[0])) and bool((lse[0] == -math.inf).all())


@pytest.mark.parametrize("lens", [[40000], [1, 9000, 30], [5000, 5001, 4999, 1]])
@pytest.mark.parametrize("H", [16, 32, 128])
@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_absorbed_long(gpu, lens, H, dtype):
    """A long axis shared by many workgroups, joined from their partial results; repeated calls give the same bits."""
    pg = _Paged(7, lens, 512, 64, dtype, page=64)
    ql, qr = _queries(4, len(lens), H, 512, 64)
    out, lse = _check_absorbed(pg, lens, ql, qr, None, 0.07)
    again = _la().absorbed_attention(ql, qr, pg.cache, pg.table, pg.lens, scale=0.07, return_lse=True)
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("H,page", [(4, 32), (33, 24), (64, 64), (128, 16)])
def test_absorbed_many_sequences(gpu, H, page, dtype):
    """More sequences than a wave has lanes, and fewer row groups than shares, more, and about as many."""
    for count in (70, 150, 290):
        lens = [(37 * b) % 450 if b % 5 else 0 for b in range(count)]
        lens[3], lens[count - 1] = 6000, 1
        pg = _Paged(count, lens, 256, 64, dtype, page=page)
        ql, qr = _queries(count, count, H, 256, 64)
        out, lse = _check_absorbed(pg, lens, ql, qr, None, 0.07)
        again = _la().absorbed_attention(ql, qr, pg.cache, pg.table, pg.lens, scale=0.07, return_lse=True)
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_absorbed_shared_page_strides(gpu, dtype):
    """A page that several table entries name, pages that lie on one another, and one row for all places of a page."""
    la = _la()
    lens = [300, 64, 129]
    ql, qr = _queries(6, 3, 16, 512, 64)
    pg = _Paged(22, [64], 512, 64, dtype, page=64)
    table = pg.table.expand(3, -1)[:, :1].expand(3, 5)
    got = la.absorbed_attention(ql, qr, pg.cache, table.contiguous(), _i32(lens), scale=0.07)
    c = la.LatentCache(*(None if t is None else t[int(pg.table[0, 0])][None].expand(5, *t.shape[1:])
                         for t in (pg.cache.latent, pg.cache.rope, pg.cache.scale)))
    order = torch.arange(5, device="cuda", dtype=torch.int32)[None].expand(3, 5).contiguous()
    assert torch.equal(la.absorbed_attention(ql, qr, c, order, _i32(lens), scale=0.07), got)
    one = la.LatentCache(*(None if t is None else t[:, :1].expand(*t.shape) for t in (pg.cache.latent, pg.cache.rope)),
                         None if pg.cache.scale is None else pg.cache.scale[:, :1].expand(*pg.cache.scale.shape).contiguous())
    full = la.LatentCache(*(None if t is None else t.contiguous() for t in (one.latent, one.rope, one.scale)))
    assert torch.equal(la.absorbed_attention(ql, qr, one, table.contiguous(), _i32(lens), scale=0.07),
                       la.absorbed_attention(ql, qr, full, table.contiguous(), _i32(lens), scale=0.07))


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("H", [8, 32, 64, 128])
def test_absorbed_growing_scores(gpu, H, dtype):
    """Each tile's scores far above the last one's, then far below: the running maximum moves tile by tile."""
    lens = [640, 640]
    pg = _Paged(11, lens, 512, 64, dtype, page=64, std=0.5)
    ql, qr = _queries(5, 2, H, 512, 64, std=0.0)
    ql, qr = ql.clone(), qr.clone()
    qr[..., 0] = 1.0
    for b, sign in ((0, 1.0), (1, -1.0)):
        j = torch.arange(640, device="cuda")
        i = pg.table[b].long()[j // 64]
        ramp = sign * (j // 64).float() * 40.0
        if dtype == BF16:
            pg.cache.rope[i, j % 64, 0] = ramp.to(BF16)
            pg.rows[b][:, 512] = ramp.to(BF16).to(ref.F64)
        else:
            s = pg.cache.scale[i, j % 64].clamp(min=1.0)
            pg.cache.scale[i, j % 64] = s
            r8 = (ramp / s).to(E4M3)
            pg.cache.rope.view(torch.uint8)[i, j % 64, 0] = r8.view(torch.uint8)
            rows = _cache_rows(pg.cache, i * 64 + j % 64)
            pg.rows[b] = rows
    _check_absorbed(pg, lens, ql, qr, None, 1.0)


def test_absorbed_huge_scores(gpu):
    """Scores in the thousands: one key takes all of the weight."""
    lens = [300]
    pg = _Paged(12, lens, 512, 64, BF16, page=64, std=8.0)
    ql, qr = _queries(6, 1, 16, 512, 64, std=30.0)
    la = _la()
    out, lse = la.absorbed_attention(ql, qr, pg.cache, pg.table, pg.lens, scale=1.0, return_lse=True)
    want, wl, _, _ = ref.absorbed(ql, qr, pg.rows, lens, [0, 1], 1.0)
    # the scores' rounding moves weight between keys that tie; the sum's logarithm is theirs either way
    ref.assert_within(lse, wl, 640 * ref.E * 576 * 8 * 30 * 4 + 1e-6 * wl.abs())
    assert torch.isfinite(out).all()


def test_absorbed_strides_and_outputs(gpu):
    la = _la()
    lens, H = [70, 10, 300], 16
    pg = _Paged(13, lens, 512, 64, BF16, page=16, joint=True)
    ql, qr = _queries(7, 3, H, 512, 64)
    want, _ = _check_absorbed(pg, lens, ql, qr, None, 0.07)
    call = lambda a, b, table=pg.table, lens=pg.lens, **kw: la.absorbed_attention(a, b, pg.cache, table, lens, scale=0.07, **kw)  # noqa: E731
    assert torch.equal(call(ql.transpose(0, 1).contiguous().transpose(0, 1), qr.contiguous()), want)
    odd = torch.zeros((3, H, 512 + 1), dtype=BF16, device="cuda")
    odd[..., 1:] = ql
    assert torch.equal(call(odd[..., 1:], qr), want)
    wide = torch.full((3, pg.table.shape[1] + 4), -5, dtype=torch.int32, device="cuda")
    wide[:, 2:-2] = pg.table
    assert torch.equal(call(ql, qr, wide[:, 2:-2]), want)
    assert torch.equal(call(ql, qr, pg.table.T.contiguous().T), want)
    lens2 = torch.stack([pg.lens, pg.lens * 0], 1)[:, 0]
    assert torch.equal(call(ql, qr, lens=lens2), want)
    out = torch.full((3, H, 514), 2.0, dtype=BF16, device="cuda")
    assert torch.equal(call(ql, qr, out=out[..., 1:513]), want)
    assert torch.equal(out[..., 1:513], want) and bool((out[..., 0] == 2).all())
    # q_latent of one row for all tokens
    one = ql[:1].expand(3, H, 512)
    assert torch.equal(call(one, qr), call(one.contiguous(), qr))


@pytest.mark.parametrize("H", [16, 128])
def test_absorbed_uncovered_tokens(gpu, H):
    """A padded batch: tokens before the first and behind the last sequence."""
    la = _la()
    lens = [70, 10]
    pg = _Paged(14, lens, 512, 64, BF16, page=16)
    ql, qr = _queries(8, 9, H, 512, 64)
    starts = _i32([1, 3, 4])
    out, lse = la.absorbed_attention(ql, qr, pg.cache, pg.table, pg.lens, scale=0.07, query_starts=starts, return_lse=True)
    want, _ = _check_absorbed(pg, lens, ql[1:4], qr[1:4], [0, 2, 3], 0.07)
    assert torch.equal(out[1:4], want)
    for t in (0, 4, 8):
        assert bool((out[t] == 0).all()) and bool((lse[t] == -math.inf).all())
    kept = torch.full_like(out, 5.0)
    _, lse2 = la.absorbed_attention(ql, qr, pg.cache, pg.table, pg.lens, scale=0.07, query_starts=starts, out=kept, return_lse=True)
    assert torch.equal(kept[1:4], want) and bool((kept[0] == 5).all()) and bool((kept[4:] == 5).all())
    assert torch.equal(lse2, lse)
    none = la.absorbed_attention(ql, qr, pg.cache, pg.table[:0], pg.lens[:0], scale=0.07, query_starts=starts[:1])
    assert bool((none == 0).all())
    assert la.absorbed_attention(ql[:0], qr[:0], pg.cache, pg.table[:0], pg.lens[:0], scale=0.07).shape == (0, H, 512)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("H", [16, 128])
def test_absorbed_bad_pages_and_lengths(gpu, H, dtype):
    """Ids outside the cache that a length reaches make their sequence NaN, no other; lengths past the table's reach
    are cut, negative ones empty."""
    la = _la()
    lens = [200, 200, 200, 200]
    pg = _Paged(15, lens, 512, 64, dtype, page=16)
    ql, qr = _queries(9, 4, H, 512, 64)
    good, _ = _check_absorbed(pg, lens, ql, qr, None, 0.07)
    table = pg.table.clone()
    table[1, 5] = pg.cache.latent.shape[0]
    table[2, 12] = -1
    table[3, 12] = -1  # past the shorter length below
    out, lse = la.absorbed_attention(ql, qr, pg.cache, table, _i32([200, 200, 200, 192]), scale=0.07, return_lse=True)
    assert torch.equal(out[0], good[0])
    assert torch.isnan(out[1:3]).all() and torch.isnan(lse[1:3]).all()
    assert torch.isfinite(out[3]).all()
    cut = la.absorbed_attention(ql, qr, pg.cache, pg.table[:, :12].contiguous(), _i32([2 ** 31 - 1, 192, 4000, -7]), scale=0.07)
    want, _, tol, _ = ref.absorbed(ql, qr, pg.rows, [192, 192, 192, 0], [0, 1, 2, 3, 4], 0.07)
    ref.assert_within(cut, want, tol)
    empty = _cache(0, 16, 512, 64, dtype)
    assert bool((la.absorbed_attention(ql, qr, empty, pg.table, pg.lens, scale=0.07) == 0).all())
    assert bool((la.absorbed_attention(ql, qr, pg.cache, pg.table[:, :0], pg.lens, scale=0.07) == 0).all())


@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_absorbed_rows_past_32_bit_offsets(gpu, dtype):
    """A cache whose last pages lie more than 2^32 bytes behind its first."""
    la = _la()
    page, pages = 64, 70000 if dtype == BF16 else 140000
    lens = [150]
    small = _Paged(16, lens, 512, 64, dtype, page=page, spare=0)
    c = la.LatentCache(*(None if t is None else torch.empty((pages, *t.shape[1:]), dtype=t.dtype, device="cuda")
                         for t in (small.cache.latent, small.cache.rope, small.cache.scale)))
    for big, t in zip((c.latent, c.rope, c.scale), (small.cache.latent, small.cache.rope, small.cache.scale)):
        if t is not None:
            big[-3:].copy_(t)
    small.cache, small.table = c, small.table + (pages - 3)
    ql, qr = _queries(10, 1, 16, 512, 64)
    out, _ = _check_absorbed(small, lens, ql, qr, None, 0.07)
    kv = _randn(1, 2, 576).to(BF16)
    last = torch.tensor([pages * page - 1, pages * page - 2], device="cuda")
    la.latent_cache_append(kv, last * 0, last, ref.rope_table(64, 2, "cuda"), c)
    assert float(_cache_rows(c, last).abs().max()) > 0.5


def test_absorbed_parts_join(gpu):
    """Results over two parts of a context, joined by their lse, give the result over all of it."""
    la = _la()
    lens, H = [700], 16
    pg = _Paged(17, lens, 512, 64, BF16, page=50)
    ql, qr = _queries(11, 1, H, 512, 64)
    whole, lse = _check_absorbed(pg, lens, ql, qr, None, 0.07)
    a, la_ = la.absorbed_attention(ql, qr, pg.cache, pg.table[:, :5].contiguous(), _i32([250]), scale=0.07, return_lse=True)
    b, lb = la.absorbed_attention(ql, qr, pg.cache, pg.table[:, 5:].contiguous(), _i32([450]), scale=0.07, return_lse=True)
    total = torch.logaddexp(la_, lb)
    joined = a.float() * (la_ - total).exp()[..., None] + b.float() * (lb - total).exp()[..., None]
    ref.assert_within(total, lse.to(ref.F64), 1e-5 + 0 * lse.to(ref.F64))
    # three bf16 results, each within twice U of the magnitudes behind it (values here are below 5)
    ref.assert_within(joined, whole.to(ref.F64), 6 * ref.U * 5 * torch.ones_like(whole, dtype=ref.F64))


# ---- expanded attention ----------------------------------------------------------------------------------------------


HEADS = [(128, 64), (128, 0), (64, 64), (64, 0)]


def _expanded_inputs(seed, new, lens, H, N, P, std=1.5):
    q = _randn(seed, sum(new), H, N + P, std=std).to(BF16)
    kv = _randn(seed + 1, sum(lens), H, 2 * N).to(BF16)
    return q, kv, (_randn(seed + 2, sum(lens), P).to(BF16) if P else None)


def _bounds(new):
    return [sum(new[:b]) for b in range(len(new) + 1)]


def _check_expanded(q, kv, kr, qs, ks, scale, causal, **kw):
    out, lse = _la().expanded_attention(q, kv, kr, _i32(qs), kv_starts=_i32(ks), scale=scale, causal=causal, return_lse=True, **kw)
    want, wl, tol, ltol = ref.expanded(q, kv, kr, qs, ks, scale, causal)
    ref.assert_within(out, want, tol, "out")
    ref.assert_within(lse, wl, ltol, "lse")
    return out, lse


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("N,P", HEADS)
@pytest.mark.parametrize("H", [1, 3, 8])
def test_expanded_matches(gpu, H, N, P, causal):
    """Lengths around the tile and the row block, empty sequences, chunks against longer contexts, and more query
    tokens than keys."""
    new = [0, 1, 63, 64, 65, 128, 129, 300, 5, 1, 17, 40]
    lens = [9, 1, 63, 64, 65, 128, 129, 300, 700, 1000, 0, 21]
    q, kv, kr = _expanded_inputs(H, new, lens, H, N, P)
    _check_expanded(q, kv, kr, _bounds(new), _bounds(lens), 0.08, causal)


@pytest.mark.parametrize("new,lens", [([1], [20000]), ([3, 150], [9000, 12000]), ([1, 1, 1], [5000, 1, 0]), ([1000], [1000])])
def test_expanded_split(gpu, new, lens):
    """Few row blocks: the key axis is shared by workgroups; repeated calls give the same bits."""
    q, kv, kr = _expanded_inputs(3, new, lens, 2, 128, 64)
    out, lse = _check_expanded(q, kv, kr, _bounds(new), _bounds(lens), 0.08, True)
    again = _la().expanded_attention(q, kv, kr, _i32(_bounds(new)), kv_starts=_i32(_bounds(lens)), scale=0.08, return_lse=True)
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)


@pytest.mark.parametrize("N,P", HEADS)
def test_expanded_growing_scores(gpu, N, P):
    new = [400, 130]
    q, kv, kr = _expanded_inputs(4, new, new, 2, N, P, std=0.5)
    q[..., 0] = 1.0
    for b, (lo, hi) in enumerate(((0, 400), (400, 530))):
        kv[lo:hi, :, 0] = ((torch.arange(hi - lo, device="cuda") // 16) * 40.0 * (1 if b == 0 else -1)).to(BF16)[:, None]
    _check_expanded(q, kv, kr, _bounds(new), _bounds(new), 1.0, True)


def test_expanded_strides_and_outputs(gpu):
    la = _la()
    new = [70, 33]
    q, kv, kr = _expanded_inputs(5, new, new, 4, 128, 64)
    st = _bounds(new)
    want, lse = _check_expanded(q, kv, kr, st, st, 0.08, True)
    call = lambda a, b, c, s=_i32(st), **kw: la.expanded_attention(a, b, c, s, scale=0.08, **kw)  # noqa: E731
    assert torch.equal(call(q, kv, kr), want)
    rows = torch.zeros((103, 576), dtype=BF16, device="cuda")  # an append's rows: the key part behind the latent
    rows[:, 512:] = kr
    assert torch.equal(call(q, kv, rows[:, 512:]), want)
    assert torch.equal(call(q.transpose(0, 1).contiguous().transpose(0, 1), kv.transpose(0, 1).contiguous().transpose(0, 1), kr), want)
    off = torch.zeros((103, 4, 257), dtype=BF16, device="cuda")
    off[..., 1:] = kv
    assert torch.equal(call(q, off[..., 1:], kr), want)
    out = torch.full((103, 4, 130), 2.0, dtype=BF16, device="cuda")
    assert torch.equal(call(q, kv, kr, out=out[..., 1:129]), want)
    assert torch.equal(out[..., 1:129], want) and bool((out[..., 129] == 2).all())
    # the same keys for all heads
    one = kv[:, :1].expand(103, 4, 256)
    assert torch.equal(call(q, one, kr), call(q, one.contiguous(), kr))
    # tokens outside the sequences
    pad = torch.cat([q[:1], q, q[:3]])
    starts = _i32([s + 1 for s in st])
    got, l2 = la.expanded_attention(pad, kv, kr, starts, kv_starts=_i32(st), scale=0.08, return_lse=True)
    assert torch.equal(got[1:104], want) and torch.equal(l2[1:104], lse)
    assert bool((got[0] == 0).all()) and bool((got[104:] == 0).all()) and bool((l2[104:] == -math.inf).all())
    kept = torch.full_like(got, 5.0)
    la.expanded_attention(pad, kv, kr, starts, kv_starts=_i32(st), scale=0.08, out=kept)
    assert torch.equal(kept[1:104], want) and bool((kept[0] == 5).all()) and bool((kept[104:] == 5).all())
    assert call(q[:0], kv[:0], kr[:0], _i32([0, 0])).shape == (0, 4, 128)
    assert bool((call(q, kv[:0], kr[:0], _i32(st), kv_starts=_i32([0, 0, 0])) == 0).all())
    assert bool((call(q, kv, kr, _i32([0])) == 0).all())


def test_expanded_keeps_to_its_sequence(gpu):
    """Keys of the next sequence, and keys that no sequence holds, may be anything."""
    la = _la()
    new = [70, 33]
    q, kv, kr = _expanded_inputs(6, new, new, 2, 128, 64)
    want, _ = _check_expanded(q, kv, kr, [0, 70, 103], [0, 70, 103], 0.08, True)
    kv2, kr2 = kv.clone(), kr.clone()
    kv2[70:], kr2[70:] = math.nan, math.inf
    got = la.expanded_attention(q[:70], kv2, kr2, _i32([0, 70]), scale=0.08)
    assert torch.equal(got, want[:70])
    # starts outside the tensors are cut to them
    cut = la.expanded_attention(q, kv, kr, _i32([0, 70, 4000]), kv_starts=_i32([-9, 70, 9999]), scale=0.08)
    assert torch.equal(cut, want)


# An average of more than 128 new tokens and 1024 keys: blocks of 256 query rows.
WIDE_NEW, WIDE_LENS = [0, 300, 1, 0, 700, 257, 64], [9, 3000, 2500, 0, 700, 257, 2600]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("N,P", HEADS)
@pytest.mark.parametrize("H", [1, 3])
def test_expanded_long_prompts(gpu, H, N, P, causal):
    q, kv, kr = _expanded_inputs(H, WIDE_NEW, WIDE_LENS, H, N, P)
    out, lse = _check_expanded(q, kv, kr, _bounds(WIDE_NEW), _bounds(WIDE_LENS), 0.08, causal)
    again = _la().expanded_attention(q, kv, kr, _i32(_bounds(WIDE_NEW)), kv_starts=_i32(_bounds(WIDE_LENS)), scale=0.08,
                                     causal=causal, return_lse=True)
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)


@pytest.mark.parametrize("new,lens", [([2200], [2140]),  # the first 60 query tokens see no key
                                      ([129], [40000]), ([1030, 250], [5000, 250]), ([2049] * 3, [2049] * 3)])
def test_expanded_long_prompt_blocks(gpu, new, lens):
    """Rows that see nothing, a key axis shared by workgroups, and more row blocks than CUs."""
    H = 12 if len(new) == 3 else 2
    q, kv, kr = _expanded_inputs(9, new, lens, H, 128, 64)
    _check_expanded(q, kv, kr, _bounds(new), _bounds(lens), 0.08, True)


@pytest.mark.parametrize("N,P", HEADS)
@pytest.mark.parametrize("sign", [1, -1])
def test_expanded_long_prompt_growing_scores(gpu, N, P, sign):
    """Scores that climb by 40 every 16 keys, past what a first tile's maximum can hold, and that fall as fast."""
    new = [2300]
    q, kv, kr = _expanded_inputs(10, new, new, 2, N, P, std=0.5)
    q[..., 0] = 1.0
    kv[:, :, 0] = ((torch.arange(2300, device="cuda") // 16) * 40.0 * sign).to(BF16)[:, None]
    _check_expanded(q, kv, kr, [0, 2300], [0, 2300], 1.0, True)


def test_expanded_long_prompt_neighbours(gpu):
    """Keys outside a sequence may be anything, in memory and left over on the chip."""
    la = _la()
    new = [2150, 40]
    q, kv, kr = _expanded_inputs(11, new, new, 4, 128, 64)
    want, _ = _check_expanded(q[:2150], kv[:2150], kr[:2150], [0, 2150], [0, 2150], 0.08, True)
    bad_kv, bad_kr = torch.full_like(kv, math.nan), torch.full_like(kr, math.inf)
    la.expanded_attention(q[:2150], bad_kv[:2150], bad_kr[:2150], _i32([0, 2150]), scale=0.08)
    kv2, kr2 = bad_kv.clone(), bad_kr.clone()
    kv2[:2150], kr2[:2150] = kv[:2150], kr[:2150]
    assert torch.equal(la.expanded_attention(q[:2150], kv2, kr2, _i32([0, 2150]), scale=0.08), want)
    # starts outside the tensors are cut to them; a caller's rows outside the sequences stay
    pad = torch.cat([q[:1], q[:2150], q[:3]])
    kept = torch.full((2154, 4, 128), 5.0, dtype=BF16, device="cuda")
    la.expanded_attention(pad, kv[:2150], kr[:2150], _i32([1, 2151]), kv_starts=_i32([-3, 9999]), scale=0.08, out=kept)
    assert torch.equal(kept[1:2151], want) and bool((kept[0] == 5).all()) and bool((kept[2151:] == 5).all())
    got, lse = la.expanded_attention(pad, kv[:2150], kr[:2150], _i32([1, 2151]), kv_starts=_i32([0, 2150]), scale=0.08,
                                     return_lse=True)
    assert torch.equal(got[1:2151], want) and bool((got[0] == 0).all()) and bool((got[2151:] == 0).all())
    assert bool((lse[0] == -math.inf).all()) and bool((lse[2151:] == -math.inf).all())


def test_expanded_long_prompt_strides(gpu):
    la = _la()
    q, kv, kr = _expanded_inputs(12, [2100], [2100], 4, 128, 64)
    st = _i32([0, 2100])
    want = la.expanded_attention(q, kv, kr, st, scale=0.08)
    heads_first = lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    rows = torch.zeros((2100, 576), dtype=BF16, device="cuda")
    rows[:, 512:] = kr
    assert torch.equal(la.expanded_attention(heads_first(q), heads_first(kv), rows[:, 512:], st, scale=0.08), want)
    one = kv[:, :1].expand(2100, 4, 256)
    assert torch.equal(la.expanded_attention(q, one, kr, st, scale=0.08),
                       la.expanded_attention(q, one.contiguous(), kr, st, scale=0.08))


@pytest.mark.parametrize("rows", [5, 150])
def test_expanded_many_sequences(gpu, rows):
    """More sequences than a wave has lanes, empty ones among them."""
    new = [(rows if b % 3 else 0) for b in range(150)] + [1]
    lens = [n + (40 if rows == 5 else 1500 * (b % 50 == 1)) for b, n in enumerate(new)]
    q, kv, kr = _expanded_inputs(13, new, lens, 1, 64, 0)
    _check_expanded(q, kv, kr, _bounds(new), _bounds(lens), 0.1, True)


def test_expanded_rows_past_32_bit_offsets(gpu):
    S, H = 70000, 128
    kv = torch.empty((S, H, 256), dtype=BF16, device="cuda")
    tail = _randn(1, 200, H, 256).to(BF16)
    kv[-200:] = tail
    q, kr = _randn(2, 5, H, 192).to(BF16), _randn(3, S, 64).to(BF16)
    got = _la().expanded_attention(q, kv, kr, _i32([0, 5]), kv_starts=_i32([S - 200, S]), scale=0.08)
    want = _la().expanded_attention(q, tail, kr[-200:].contiguous(), _i32([0, 5]), kv_starts=_i32([0, 200]), scale=0.08)
    full, _, tol, _ = ref.expanded(q[:, :3], tail[:, :3], kr[-200:], [0, 5], [0, 200], 0.08, True)
    ref.assert_within(want[:, :3], full, tol)
    ref.assert_within(got.float(), want.to(ref.F64), 2 * ref.U * 5 * torch.ones_like(want, dtype=ref.F64))


# ---- together -----------------------------------------------------------------------------------------------------------


class _Layer:
    """A latent-attention layer's weights and one prompt batch, run through the framework's calls."""

    def __init__(self, H=8, hidden=512, dtype=BF16):
        from fused_cpp_amd import deepseek_v4_w8a8 as ds

        la = _la()
        self.H, self.N, self.P, self.R = H, 128, 64, 512
        lin = lambda s, n, k: ds.prepare_deepseek_v4_w8a8_linear_weight(_randn(s, n, k, std=k ** -0.5).to(BF16))  # noqa: E731
        self.wq, self.wkv, self.wo = lin(1, H * 192, hidden), lin(2, 576, hidden), lin(3, hidden, H * 128)
        kv_b = _randn(4, H, 256, 512, std=512 ** -0.5).to(BF16)
        self.kv_b = kv_b
        self.w_uk = la.prepare_head_projection(kv_b[:, :128].transpose(1, 2))
        self.w_uv = la.prepare_head_projection(kv_b[:, 128:])
        self.up = la.prepare_head_projection(kv_b)
        self.kv_norm = (1 + 0.1 * _randn(5, 512)).to(BF16)
        self.table = ref.rope_table(64, 512, "cuda")
        self.scale = 192 ** -0.5
        self.cache = la.allocate_latent_cache(40, 16, dtype=dtype)

    def queries(self, x, pos):
        from fused_cpp_amd import deepseek_v4_w8a8 as ds

        q = ds.deepseek_v4_w8a8_linear(x, self.wq).view(-1, self.H, 192)
        return _la().head_norm_rope(q, pos, self.table, normalize=False, out=q)

    def append(self, x, pos, slots):
        from fused_cpp_amd import deepseek_v4_w8a8 as ds

        return _la().latent_cache_append(ds.deepseek_v4_w8a8_linear(x, self.wkv), pos, slots, self.table, self.cache,
                                         weight=self.kv_norm, return_rows=True)

    def prefill(self, x, pos, slots, starts):
        la = _la()
        q, rows = self.queries(x, pos), self.append(x, pos, slots)
        up = la.head_projection(rows[:, None, :512].expand(-1, self.H, -1), self.up)
        return la.expanded_attention(q, up, rows[:, 512:], starts, scale=self.scale), (q, rows, up)

    def decode(self, x, pos, slots, table, lens, starts=None):
        la = _la()
        q = self.queries(x, pos)
        self.append(x, pos, slots)
        ql = la.head_projection(q[..., :128], self.w_uk)
        o = la.absorbed_attention(ql, q[..., 128:], self.cache, table, lens, scale=self.scale, query_starts=starts)
        return la.head_projection(o, self.w_uv), (q, ql, o)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_layer_prefill_then_decode(gpu, dtype):
    """Prompts through the expanded form into the cache, then tokens through the absorbed form over it: each step
    against the formulas on the inputs it got, and the two forms of one layer against each other."""
    from fused_cpp_amd import deepseek_v4_w8a8 as ds

    layer = _Layer(dtype=dtype)
    H, new = layer.H, [37, 5, 100]
    st = _bounds(new)
    x = _randn(20, sum(new), 512).to(BF16)
    pos = torch.cat([torch.arange(n) for n in new]).cuda()
    order = torch.randperm(40, generator=torch.Generator().manual_seed(1)).int()
    table = order[:30].view(3, 10).cuda()
    slots = torch.cat([table[b].long()[torch.arange(n, device="cuda") // 16] * 16 + torch.arange(n, device="cuda") % 16
                       for b, n in enumerate(new)])
    values, (q, rows, up) = layer.prefill(x, pos, slots, _i32(st))
    want, _, tol, _ = ref.expanded(q, up, rows[:, 512:], st, st, layer.scale, True)
    ref.assert_within(values, want, tol)
    assert ds.deepseek_v4_wo_b_w8a8(values.view(-1, H * 128), layer.wo).shape == (sum(new), 512)
    # the absorbed form over the same cache, all prompt tokens as queries
    again, (_, ql, o) = layer.decode(x, pos, slots, table, _i32(new), _i32(st))
    cached = [_cache_rows(layer.cache, slots[a:b]) for a, b in zip(st, st[1:])]
    want, _, tol, _ = ref.absorbed(ql, q[..., 128:], cached, new, st, layer.scale)
    ref.assert_within(o, want, tol)
    cos = torch.nn.functional.cosine_similarity(again.float().flatten(), values.float().flatten(), 0)
    # relative error of each side's rounded inputs: bf16 2^-8, cached e4m3 rows 2^-4; 1 - cos is half its square
    assert 1 - float(cos) < (0.5 * (8 * ref.U) ** 2 if dtype == BF16 else 0.5 * (4 * 2.0 ** -4) ** 2)
    # three decode steps of one token a sequence
    lens = list(new)
    for step in range(3):
        xt = _randn(30 + step, 3, 512).to(BF16)
        p = torch.tensor(lens, device="cuda")
        s = table.long()[torch.arange(3, device="cuda"), p // 16] * 16 + p % 16
        lens = [n + 1 for n in lens]
        _, (qd, ql, o) = layer.decode(xt, p, s, table, _i32(lens))
        cached = [_cache_rows(layer.cache, table[b].long()[torch.arange(n, device="cuda") // 16] * 16 +
                              torch.arange(n, device="cuda") % 16) for b, n in enumerate(lens)]
        want, _, tol, _ = ref.absorbed(ql, qd[..., 128:], cached, lens, [0, 1, 2, 3], layer.scale)
        ref.assert_within(o, want, tol)


def test_layer_captured(gpu):
    """A decode step captured once and replayed for growing lengths, with eager work and other graphs in between."""
    layer, eager = _Layer(), _Layer()
    eager.cache.latent.copy_(layer.cache.latent)
    B = 3
    table = torch.arange(30, dtype=torch.int32).view(3, 10).cuda()
    x, pos, slots = torch.zeros((B, 512), dtype=BF16, device="cuda"), torch.zeros(B, dtype=torch.long, device="cuda"), torch.full((B,), -1, device="cuda")
    lens = _i32([1, 1, 1])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        layer.decode(x, pos, slots, table, lens)
    torch.cuda.current_stream().wait_stream(s)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(layer.decode(x, pos, slots, table, lens)[0])
        graphs.append(g)
    layer.cache.latent.zero_()
    layer.cache.rope.zero_()
    for step, n in enumerate([0, 1, 63, 64, 100, 101, 159]):
        x.copy_(_randn(40 + step, B, 512).to(BF16))
        pos.fill_(n)
        slots.copy_(table.long()[:, n // 16] * 16 + n % 16)
        lens.fill_(n + 1)
        want = eager.decode(x, pos, slots, table, lens)[0]
        for g, o in zip(graphs, outs):
            o.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(o, want), step
        _randn(1, 1000, 1000) @ _randn(2, 1000, 1000)


def test_prefill_captured(gpu):
    la = _la()
    new = [100, 30]
    q, kv, kr = _expanded_inputs(7, new, new, 4, 128, 64)
    starts = _i32([0, 100, 130])
    la.expanded_attention(q, kv, kr, starts, scale=0.08)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = la.expanded_attention(q, kv, kr, starts, scale=0.08)
    for split in (100, 1, 130, 64, 0):
        starts.copy_(_i32([0, split, 130]))
        want = la.expanded_attention(q, kv, kr, starts, scale=0.08)
        out.fill_(9)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), split


def test_side_streams(gpu):
    """Calls on two streams at once, on tensors of another stream, give what they give alone."""
    la = _la()
    lens = [3000, 50]
    pg = _Paged(21, lens, 512, 64, BF16, page=64)
    ql, qr = _queries(12, 2, 16, 512, 64)
    q, kv, kr = _expanded_inputs(8, [3], [4000], 4, 128, 64)
    st, kst = _i32([0, 3]), _i32([0, 4000])
    a = la.absorbed_attention(ql, qr, pg.cache, pg.table, pg.lens, scale=0.07)
    b = la.expanded_attention(q, kv, kr, st, kv_starts=kst, scale=0.08)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append((la.absorbed_attention(ql, qr, pg.cache, pg.table, pg.lens, scale=0.07),
                        la.expanded_attention(q, kv, kr, st, kv_starts=kst, scale=0.08)))
    torch.cuda.synchronize()
    for x, y in got:
        assert torch.equal(x, a) and torch.equal(y, b)
