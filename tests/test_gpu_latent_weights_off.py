"""GPU weights of cached tokens where a query's lse of -inf turns it off: it adds nothing, whatever its row holds."""

from __future__ import annotations

import math

import pytest
import torch

from tests.test_gpu_latent_attention import BF16, E4M3, _i32, _la, _Paged, _queries
from tests.test_gpu_latent_context import _lc, _starts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("H,new", [(1, [1, 1, 1]), (16, [1, 1, 1]), (5, [3, 9, 1]), (128, [1, 1, 1]), (16, [40, 3, 33]), (128, [20, 32, 5])])
@pytest.mark.parametrize("off", [math.nan, math.inf, -math.inf, 3.0e38])
def test_rows_that_are_off_may_hold_anything(gpu, H, new, dtype, off):
    """The first, the last (which fills a chunk's places behind it) and some heads of the query rows."""
    lens = [300, 130, 64]
    pg = _Paged(7, lens, 512, 64, dtype, page=16)
    T = sum(new)
    ql, qr = _queries(5, T, H, 512, 64)
    st = _i32(_starts(new))
    _, lse = _la().absorbed_attention(ql, qr, pg.cache, pg.table, pg.lens, scale=0.07, query_starts=st, return_lse=True)
    mine = torch.zeros((T, H), dtype=torch.bool)
    mine[0], mine[-1], mine[T // 2, ::3], mine[new[0] - 1, H - 1] = True, True, True, True
    mine = mine.cuda()
    lse = lse.masked_fill(mine, -math.inf)
    previous = torch.rand((3, 320), device="cuda")

    def weights(q, r):
        return _lc().attention_weights(q, r, pg.cache, pg.table, pg.lens, lse, scale=0.07, query_starts=st, previous=previous)

    want = weights(ql, qr)
    assert bool(torch.isfinite(want).all())
    bad, rest = ql.masked_fill(mine[..., None], off), qr.masked_fill(mine[..., None], off)
    assert torch.equal(weights(bad, rest), want)
    assert torch.equal(weights(bad, qr), want) and torch.equal(weights(ql, rest), want)
