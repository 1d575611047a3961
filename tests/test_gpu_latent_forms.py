"""Every form of the latent operators' kernels, at sizes that leave remainders in it. Which form a size takes follows
from rules on sizes in the kernels' sources; they are restated here, so that a case that no longer reaches its form fails."""

from __future__ import annotations

import pytest
import torch

from tests import latent_reference as ref
from tests.test_gpu_latent_attention import BF16, E4M3, _check_absorbed, _check_norm_rope, _la, _Paged, _queries, _randn

pytestmark = pytest.mark.gpu


def _tiles(n, of):
    return -(-n // of)


# ---- per-head products -------------------------------------------------------------------------------------------------


def _projection_tile(T, H, N):
    """Tokens and channels of a wave's tile, in sixteens: the largest that gives each of 1024 SIMDs a wave."""
    for mt, nt, least in ((4, 8, 33), (4, 4, 33), (2, 4, 33), (2, 2, 17)):
        if T >= least and _tiles(T, 16 * mt) * H * _tiles(_tiles(N, 16), nt) >= 1024:
            return mt, nt
    return 1, 1


@pytest.mark.parametrize("tile,T,H,N,K", [
    ((1, 1), 16, 128, 512, 128), ((1, 1), 33, 32, 136, 40), ((1, 1), 300, 3, 72, 520),
    ((2, 2), 17, 128, 512, 128), ((2, 2), 31, 128, 264, 136), ((2, 2), 64, 128, 128, 512), ((2, 2), 97, 47, 200, 72),
    ((2, 4), 49, 96, 512, 128), ((2, 4), 33, 100, 520, 40), ((2, 4), 113, 128, 136, 520), ((2, 4), 180, 128, 72, 8),
    ((4, 4), 33, 128, 512, 128), ((4, 4), 47, 128, 512, 128), ((4, 4), 48, 128, 512, 128), ((4, 4), 300, 128, 128, 512),
    ((4, 4), 65, 97, 328, 200),
    ((4, 8), 300, 128, 512, 128), ((4, 8), 513, 128, 128, 512), ((4, 8), 2047, 32, 128, 136), ((4, 8), 500, 128, 136, 520),
    ((4, 8), 77, 128, 520, 24),
])
def test_projection_tiles(gpu, tile, T, H, N, K):
    assert _projection_tile(T, H, N) == tile
    la = _la()
    w = _randn(N, H, N, K).to(BF16)
    x = _randn(K, T, H, K + 8).to(BF16)[..., :K]
    wide = torch.full((T, H, N + 4), 3.0, dtype=BF16, device="cuda")
    got = la.head_projection(x, la.prepare_head_projection(w), out=wide[..., :N])
    assert bool((wide[..., N:] == 3).all())
    for h in sorted({0, 1, H // 2, H - 1}):
        a, b = x[:, h].to(ref.F64), w[h].to(ref.F64).T.contiguous()
        ref.assert_within(got[:, h], a @ b, ref.U * (a @ b).abs() + K * ref.E * (a.abs() @ b.abs()), (tile, h))
    # the other heads by fp32 products of the same operands, each side within its bound
    want = torch.bmm(x.float().transpose(0, 1).contiguous(), w.float().transpose(1, 2).contiguous()).transpose(0, 1)
    mag = torch.bmm(x.float().abs().transpose(0, 1).contiguous(), w.float().abs().transpose(1, 2).contiguous()).transpose(0, 1)
    ref.assert_within(got, want.to(ref.F64), ref.U * want.abs().to(ref.F64) + 3 * K * ref.E * mag.to(ref.F64))


def test_projection_of_one_input_for_all_heads(gpu):
    """The up-projection of a prompt's latent rows: one x a token, read by every head."""
    la = _la()
    w = la.prepare_head_projection(_randn(1, 128, 256, 512).to(BF16))
    x = _randn(2, 150, 576).to(BF16)
    assert torch.equal(la.head_projection(x[:, None, :512].expand(-1, 128, -1), w),
                       la.head_projection(x[:, None, :512].expand(-1, 128, -1).contiguous(), w))


# ---- norm and rotation, two row groups in flight ------------------------------------------------------------------------


def _two_groups(rows, D):
    """Rows a workgroup takes at a time, and whether it takes two such groups: from 32768 groups up."""
    lanes = next(n for n in (8, 16, 32, 64) if D // 8 <= n or n == 64)
    return 256 // lanes, rows >= 256 // lanes * 32768


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("T,H,D,P", [
    (1048577, 1, 64, 32),   # one row in the last workgroup's first group, none in its second
    (349540, 3, 48, 48),    # 1048620 rows: its second group in part
    (174770, 3, 128, 64), (87385, 3, 192, 64), (52431, 5, 256, 128), (21847, 6, 512, 64), (43691, 3, 576, 64), (131075, 1, 1024, 64)])
def test_norm_rope_two_groups(gpu, T, H, D, P, interleaved, in_place):
    assert _two_groups(T * H, D)[1]
    x = _randn(T + D, T, H, D, std=3.0).to(BF16)
    table = ref.rope_table(P, 1000, "cuda")
    pos = torch.randint(-1, 1000, (T,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(T)).clamp(min=0)
    w = (1 + 0.2 * _randn(D, D)).to(BF16)
    for weight, normalize, inverse in ((w, True, False), (None, False, True)):
        want = _check_norm_rope(x, pos, table, weight, normalize, inverse, interleaved, 1e-6)
        if in_place:
            wide = torch.zeros((T, H, D + 8), dtype=BF16, device="cuda")
            y = wide[..., :D]
            y.copy_(x)
            _la().head_norm_rope(y, pos, table, weight=weight, normalize=normalize, inverse=inverse, interleaved=interleaved, out=y)
            assert torch.equal(y, want) and bool((wide[..., D:] == 0).all())


@pytest.mark.parametrize("interleaved", [True, False])
def test_norm_rope_two_groups_one_short(gpu, interleaved):
    """Just below the limit: one group."""
    assert not _two_groups(131071, 512)[1] and _two_groups(131072, 512)[1]
    for T in (131071, 131072):
        x, pos = _randn(T, T, 1, 512).to(BF16), torch.arange(T, device="cuda") % 50
        _check_norm_rope(x, pos, ref.rope_table(64, 50, "cuda"), None, True, False, interleaved, 1e-6)


# ---- absorbed attention: joining partial results ------------------------------------------------------------------------


def _join_form(count, H, n, R, e4m3, cus):
    """Rows of a group, and whether a strip's partial results are spread over many workgroups."""
    per = n * H
    rows = next(r for r in (16, 32, 64, 128) if per <= r or r == 128)
    groups = count * n * H // rows + count
    shares = cus // 2 if rows == 128 else cus * (2 if e4m3 and rows == 16 else 1)
    return rows, min(groups, shares) * (rows // 16) * (R // 4) <= 512


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("R,P", [(512, 64), (512, 0), (256, 64), (256, 0)])
@pytest.mark.parametrize("rows,H,n,count,spread_from", [
    (16, 16, 1, 1, 512), (16, 16, 1, 2, 512), (16, 9, 1, 4, 256), (16, 16, 1, 3, 256), (16, 16, 1, 40, 0), (16, 5, 3, 150, 0),
    (32, 32, 1, 1, 512), (32, 17, 1, 1, 512), (32, 32, 1, 2, 256), (32, 16, 2, 20, 0),
    (64, 33, 1, 1, 512), (64, 64, 1, 1, 256), (64, 33, 1, 30, 0),
    (128, 65, 1, 1, 256), (128, 128, 1, 1, 0), (128, 128, 1, 33, 0), (128, 33, 3, 70, 0)])
def test_absorbed_joins(gpu, rows, H, n, count, spread_from, R, P, e4m3):
    """Long sequences among short ones, so that groups end up with one, a few and many shares."""
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    assert _join_form(count, H, n, R, e4m3, cus) == (rows, R <= spread_from)  # latent widths whose joins are spread
    lens = [(37 * b) % 300 if b % 4 else 0 for b in range(count)]
    lens[-1], lens[0] = 3001, 9000
    pg = _Paged(count, lens, R, P, E4M3 if e4m3 else BF16, page=48)
    ql, qr = _queries(count, n * count, H, R, P)
    starts = [n * b for b in range(count + 1)]
    out, lse = _check_absorbed(pg, lens, ql, qr, starts, 0.07)
    again = _la().absorbed_attention(ql, qr, pg.cache, pg.table, pg.lens, scale=0.07, return_lse=True,
                                     query_starts=torch.tensor(starts, dtype=torch.int32, device="cuda"))
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)
