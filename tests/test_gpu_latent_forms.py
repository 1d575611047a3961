"""Every form of the latent operators' kernels, at sizes that leave remainders in it. Which form a size takes follows
from rules on sizes in the kernels' sources; they are restated here, so that a case that no longer reaches its form fails."""

from __future__ import annotations

import pytest
import torch

from tests import latent_reference as ref
from tests.test_gpu_latent_attention import BF16, _check_norm_rope, _la, _randn

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
