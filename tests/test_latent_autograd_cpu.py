"""Forward-mode tangents are refused like gradients: no operator passes one on (host tensors reach the check)."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd

from fused_cpp_amd import latent_attention as la

BF16 = torch.bfloat16


def _z(*shape, dtype=BF16):
    return torch.zeros(shape, dtype=dtype)


def _i(*shape):
    return torch.zeros(shape, dtype=torch.int32)


TABLE = _z(8, 64, dtype=torch.float32)
CACHE = la.allocate_latent_cache(4, 16, device="cpu")
CALLS = {
    "head_norm_rope": (la.head_norm_rope, dict(x=_z(3, 2, 192), positions=_i(3), cos_sin=TABLE, weight=_z(192), out=_z(3, 2, 192))),
    "latent_cache_append": (la.latent_cache_append, dict(kv=_z(3, 576), positions=_i(3), slots=_i(3), cos_sin=TABLE, cache=CACHE,
                                                        weight=_z(512))),
    "prepare_head_projection": (la.prepare_head_projection, dict(weight=_z(2, 16, 16))),
    "head_projection": (la.head_projection, dict(x=_z(3, 2, 16), out=_z(3, 2, 16),
                                                 weight=la.PreparedHeadProjection(torch.zeros((2, 1024), dtype=torch.int8), 2, 16, 16))),
    "absorbed_attention": (la.absorbed_attention, dict(q_latent=_z(3, 4, 512), q_rope=_z(3, 4, 64), cache=CACHE, page_table=_i(3, 5),
                                                       kv_lens=_i(3), scale=0.1, out=_z(3, 4, 512))),
    "expanded_attention": (la.expanded_attention, dict(q=_z(5, 4, 192), kv=_z(7, 4, 256), k_rope=_z(7, 64), query_starts=_i(3),
                                                       scale=0.1, out=_z(5, 4, 128))),
}
CASES = [(name, arg) for name, (_, kw) in CALLS.items() for arg, v in kw.items()
         if isinstance(v, torch.Tensor) and v.is_floating_point()]


@pytest.mark.parametrize("name,arg", CASES)
def test_tangents_are_refused(name, arg):
    fn, kw = CALLS[name]
    with fwd.dual_level():
        dual = fwd.make_dual(kw[arg], torch.ones_like(kw[arg]))
        with pytest.raises(RuntimeError, match="tangent"):
            fn(**{**kw, arg: dual})
        with torch.no_grad(), pytest.raises(RuntimeError, match="tangent"):  # which leaves forward mode on
            fn(**{**kw, arg: dual})
    with pytest.raises(ValueError, match="device"):
        fn(**kw)


def test_cache_tangents_are_refused():
    with fwd.dual_level():
        for part in ("latent", "rope"):
            t = getattr(CACHE, part)
            cache = la.LatentCache(**{"latent": CACHE.latent, "rope": CACHE.rope, part: fwd.make_dual(t, torch.ones_like(t))})
            for name in ("latent_cache_append", "absorbed_attention"):
                fn, kw = CALLS[name]
                with pytest.raises(RuntimeError, match="tangent"):
                    fn(**{**kw, "cache": cache})
