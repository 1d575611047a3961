"""GPU absorbed attention with windows and first tokens past all contexts, to 63 bits, against the formulas in 64 bits."""

from __future__ import annotations

import pytest

from tests import context_reference as cref
from tests import latent_reference as ref
from tests.test_gpu_latent_attention import BF16, E4M3, _i32, _la, _Paged, _queries
from tests.test_gpu_latent_context import _starts

pytestmark = pytest.mark.gpu

LENS = [700, 64, 0, 3000]


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("H,n", [(16, 1), (8, 3), (64, 1), (128, 2)])
@pytest.mark.parametrize("window,sinks", [(3000, 0), (5000, 17), (2 ** 31 - 1, 2 ** 31 - 1), (2 ** 31, 2 ** 31), (2 ** 40, 2 ** 35),
                                          (2 ** 63 - 1, 2 ** 63 - 1), (7, 2 ** 40)])
def test_a_window_past_the_context_is_none(gpu, window, sinks, H, n, dtype):
    """Row groups of 16, 32, 64 and 128: output and lse are the causal ones (with all tokens first ones, too)."""
    pg = _Paged(9, LENS, 512, 64, dtype, page=64)
    ql, qr = _queries(7, 4 * n, H, 512, 64)
    st = _starts([n] * 4)
    keeps = [cref.seen_by_window(n, L, L + n, 0) for L in LENS]
    want, wl, tol, ltol = cref.absorbed(ql, qr, pg.rows, st, 0.07, keeps)
    out, lse = _la().absorbed_attention(ql, qr, pg.cache, pg.table, pg.lens, scale=0.07, query_starts=_i32(st), window=window,
                                        sinks=sinks, return_lse=True)
    ref.assert_within(out, want, tol, "out")
    ref.assert_within(lse, wl, ltol, "lse")
