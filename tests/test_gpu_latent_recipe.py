"""GPU: the steps that fused_cpp_amd.latent_context's docstring gives for a cache that is cut down, run as they stand there."""

from __future__ import annotations

import re

import pytest
import torch

from tests import context_reference as cref
from tests import latent_reference as ref
from tests.test_gpu_latent_attention import BF16, E4M3, _la, _Paged, _queries
from tests.test_gpu_latent_context import _lc

pytestmark = pytest.mark.gpu


def _steps():
    doc = _lc().__doc__
    lines = re.findall(r"^    (\S.*)$", doc[doc.index("a cache that keeps"):], re.M)
    code = "\n".join(lines).replace("absorbed_attention(...", "absorbed_attention(q_latent, q_rope, cache, page_table, kv_lens, scale=scale")
    return code.replace("scale=...", "scale=scale")


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("keep", [132, 200, 640, 700])
def test_weights_move_with_their_rows(gpu, keep, dtype):
    """Fewer, as many and more rows than the weights have columns: every kept row's sum lies at its new place, all others
    are 0, and the next step adds to the right ones."""
    lens, H, scale, columns = [600, 40, 333], 16, 0.07, 640
    pg = _Paged(41, lens, 512, 64, dtype, page=16)
    ql, qr = _queries(12, 3, H, 512, 64)
    before = torch.rand((3, columns), device="cuda")
    for b, L in enumerate(lens):
        before[b, L:] = 0
    names = {"q_latent": ql, "q_rope": qr, "cache": pg.cache, "page_table": pg.table, "kv_lens": pg.lens, "scale": scale, "keep": keep,
             "weights": before.clone(), "absorbed_attention": _la().absorbed_attention}
    names.update({n: getattr(_lc(), n) for n in _lc().__all__})
    _, lse = _la().absorbed_attention(ql, qr, pg.cache, pg.table, pg.lens, scale=scale, return_lse=True)
    total = _lc().attention_weights(ql, qr, pg.cache, pg.table, pg.lens, lse, scale=scale, previous=before)
    exec(_steps(), names)  # noqa: S102
    weights, kept = names["weights"], names["kept"].tolist()
    assert weights.shape == (3, columns)
    rows = []
    for b, L in enumerate(lens):
        stay = cref.heaviest(total[b].cpu().tolist(), L, keep, 4, 128)
        assert kept[b] == len(stay)
        assert torch.equal(weights[b, :len(stay)], total[b, stay]) and not bool(weights[b, len(stay):].any())
        rows.append(pg.rows[b][stay])
    ql, qr = _queries(13, 3, H, 512, 64)
    _, lse = _la().absorbed_attention(ql, qr, pg.cache, pg.table, names["kept"], scale=scale, return_lse=True)
    got = _lc().attention_weights(ql, qr, pg.cache, pg.table, names["kept"], lse, scale=scale, previous=weights)
    want, tol = cref.weights(ql, qr, rows, kept, [0, 1, 2, 3], lse, scale, columns, weights)
    ref.assert_within(got, want, tol)
