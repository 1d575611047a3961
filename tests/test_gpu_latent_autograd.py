"""A tensor that an operator writes counts as changed: a graph that saved it refuses to go back through it."""

from __future__ import annotations

import pytest
import torch

from tests import latent_reference as ref
from tests.test_gpu_latent_attention import BF16, E4M3, _cache, _expanded_inputs, _i32, _la, _Paged, _queries, _randn

pytestmark = pytest.mark.gpu


def _refuses_to_go_back(saved, write):
    """`write` writes to `saved`, which a product with a leaf has kept for its gradient."""
    leaf = torch.ones_like(saved, dtype=torch.float32).requires_grad_()
    y = (leaf * saved).sum()
    before = saved._version
    write()
    assert saved._version > before
    with pytest.raises(RuntimeError, match="inplace operation"):
        y.backward()


def test_outputs_count_as_changed(gpu):
    la = _la()
    table, pos = ref.rope_table(64, 50, "cuda"), torch.arange(5, device="cuda")
    x = _randn(1, 5, 4, 192).to(BF16)
    out = torch.zeros_like(x)
    _refuses_to_go_back(out, lambda: la.head_norm_rope(x, pos, table, out=out))
    _refuses_to_go_back(x, lambda: la.head_norm_rope(x, pos, table, out=x))
    wide = torch.zeros((5, 4, 400), dtype=BF16, device="cuda")  # through a view, of which the rest counts as well
    _refuses_to_go_back(wide, lambda: la.head_norm_rope(x, pos, table, out=wide[..., :192]))
    _refuses_to_go_back(wide, lambda: la.head_norm_rope(x, pos, table, out=wide[..., :384:2]))
    w = la.prepare_head_projection(_randn(2, 4, 128, 192).to(BF16))
    _refuses_to_go_back(wide, lambda: la.head_projection(x, w, out=wide[..., :128]))
    pg = _Paged(3, [70, 10], 512, 64, BF16, page=16)
    ql, qr = _queries(7, 2, 16, 512, 64)
    o = torch.zeros((2, 16, 512), dtype=BF16, device="cuda")
    _refuses_to_go_back(o, lambda: la.absorbed_attention(ql, qr, pg.cache, pg.table, pg.lens, scale=0.07, out=o))
    q, kv, kr = _expanded_inputs(5, [70], [70], 4, 128, 64)
    v = torch.zeros((70, 4, 128), dtype=BF16, device="cuda")
    _refuses_to_go_back(v, lambda: la.expanded_attention(q, kv, kr, _i32([0, 70]), scale=0.08, out=v))


@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_a_cache_counts_as_changed(gpu, dtype):
    la = _la()
    c = _cache(3, 16, 512, 64, dtype)
    kv, pos = _randn(1, 3, 576).to(BF16), torch.arange(3, device="cuda")
    table = ref.rope_table(64, 50, "cuda")
    append = lambda: la.latent_cache_append(kv, pos, pos, table, c)  # noqa: E731
    if dtype == BF16:
        _refuses_to_go_back(c.latent, append)
        _refuses_to_go_back(c.rope, append)
    else:
        before = [t._version for t in (c.latent, c.rope, c.scale)]
        append()
        assert all(t._version > b for t, b in zip((c.latent, c.rope, c.scale), before))
        _refuses_to_go_back(c.scale, append)


def test_inference_tensors(gpu):
    """Tensors made in inference mode have no version to count."""
    la = _la()
    table, pos = ref.rope_table(64, 50, "cuda"), torch.arange(5, device="cuda")
    x = _randn(1, 5, 4, 192).to(BF16)
    want = la.head_norm_rope(x, pos, table)
    with torch.inference_mode():
        out = torch.zeros_like(x)
        assert torch.equal(la.head_norm_rope(x, pos, table, out=out), want)
        c = _cache(3, 16, 512, 64, BF16)
        la.latent_cache_append(_randn(1, 3, 576).to(BF16), pos[:3], pos[:3], table, c)
    assert torch.equal(la.head_norm_rope(x, pos, table, out=out), want)
