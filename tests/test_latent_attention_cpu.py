"""Latent attention without a GPU: refusals (dtypes, shapes, values, gradients and devices are checked before any
device work), the C ABI's argument checks, and the ctypes mirror of its structures."""

from __future__ import annotations

import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

from fused_cpp_amd import cabi
from fused_cpp_amd import latent_attention as la

REPO = Path(__file__).resolve().parent.parent
BF16 = torch.bfloat16


def _z(*shape, dtype=BF16):
    return torch.zeros(shape, dtype=dtype)


def _i(*shape, dtype=torch.int32):
    return torch.zeros(shape, dtype=dtype)


def _cache(R=512, P=64, dtype=BF16, pages=4, page=16):
    return la.allocate_latent_cache(pages, page, latent_dim=R, rope_dim=P, dtype=dtype, device="cpu")


def test_public_names():
    import fused_cpp_amd

    assert "latent_attention" in fused_cpp_amd.__all__
    assert set(la.__all__) == {"LatentCache", "PreparedHeadProjection", "absorbed_attention", "allocate_latent_cache",
                               "expanded_attention", "head_norm_rope", "head_projection", "latent_cache_append",
                               "prepare_head_projection"}


def test_allocate_cache():
    c = _cache(dtype=torch.float8_e4m3fn)
    assert c.latent.shape == (4, 16, 512) and c.rope.shape == (4, 16, 64) and c.scale.shape == (4, 16)
    assert c.latent.dtype == torch.float8_e4m3fn and bool((c.latent.float() == 0).all())
    assert _cache(P=0).rope is None and _cache().scale is None
    for kw in ({"latent_dim": 384}, {"rope_dim": 32}):
        with pytest.raises(ValueError):
            la.allocate_latent_cache(1, 1, device="cpu", **kw)
    with pytest.raises(ValueError):
        la.allocate_latent_cache(1, 0, device="cpu")
    with pytest.raises(TypeError):
        la.allocate_latent_cache(1, 1, dtype=torch.float16, device="cpu")


NORM = dict(x=_z(3, 2, 192), positions=_i(3), cos_sin=_z(8, 64, dtype=torch.float32))


@pytest.mark.parametrize("error,change", [
    (TypeError, {"x": _z(3, 2, 192, dtype=torch.float32)}),
    (TypeError, {"x": _z(3, 2, 192, dtype=torch.float16)}),
    (ValueError, {"x": _z(3, 192)}),
    (ValueError, {"x": _z(3, 0, 192)}),
    (TypeError, {"positions": _i(3, dtype=torch.int16)}),
    (TypeError, {"positions": _z(3, dtype=torch.float32)}),
    (ValueError, {"positions": _i(4)}),
    (ValueError, {"positions": _i(3, 1)}),
    (TypeError, {"cos_sin": _z(8, 64)}),
    (ValueError, {"cos_sin": _z(8, 63, dtype=torch.float32)}),
    (ValueError, {"cos_sin": _z(8, 256, dtype=torch.float32)}),
    (ValueError, {"cos_sin": _z(64, dtype=torch.float32)}),
    (ValueError, {"eps": -1.0}),
    (ValueError, {"eps": float("nan")}),
    (TypeError, {"weight": _z(192, dtype=torch.float32)}),
    (ValueError, {"weight": _z(191)}),
    (ValueError, {"weight": _z(192), "normalize": False}),
    (TypeError, {"out": _z(3, 2, 192, dtype=torch.float32)}),
    (ValueError, {"out": _z(3, 2, 191)}),
    (RuntimeError, {"out": _z(3, 1, 192).expand(3, 2, 192)}),
    (RuntimeError, {"x": _z(3, 2, 192).requires_grad_()}),
    (RuntimeError, {"out": _z(3, 2, 192).requires_grad_()}),
    (ValueError, {}),  # host tensors
])
def test_norm_rope_refusals(error, change):
    with pytest.raises(error):
        la.head_norm_rope(**{**NORM, **change})


def test_norm_rope_refuses_partial_overlap():
    both = _z(2, 3, 2, 192)
    flat = both.view(-1)
    with pytest.raises(RuntimeError, match="overlap"):
        la.head_norm_rope(both[0], NORM["positions"], NORM["cos_sin"], out=flat[192:192 + 3 * 2 * 192].view(3, 2, 192))


def test_gradients_are_refused_only_while_recorded():
    x = _z(3, 2, 192).requires_grad_()
    with pytest.raises(RuntimeError, match="gradient"):
        la.head_norm_rope(**{**NORM, "x": x})
    with torch.no_grad(), pytest.raises(ValueError, match="device"):
        la.head_norm_rope(**{**NORM, "x": x})


APPEND = dict(kv=_z(3, 576), positions=_i(3), slots=_i(3), cos_sin=_z(8, 64, dtype=torch.float32))


@pytest.mark.parametrize("error,change", [
    (TypeError, {"kv": _z(3, 576, dtype=torch.float32)}),
    (ValueError, {"kv": _z(3, 575)}),
    (ValueError, {"kv": _z(576)}),
    (TypeError, {"slots": _i(3, dtype=torch.int8)}),
    (ValueError, {"slots": _i(2)}),
    (ValueError, {"positions": _i(2)}),
    (ValueError, {"cos_sin": _z(8, 32, dtype=torch.float32)}),
    (TypeError, {"weight": _z(512, dtype=torch.float32)}),
    (ValueError, {"weight": _z(576)}),
    (ValueError, {"eps": float("inf")}),
    (TypeError, {"cache": la.LatentCache(_z(4, 16, 512, dtype=torch.float16), _z(4, 16, 64, dtype=torch.float16))}),
    (ValueError, {"cache": la.LatentCache(_z(4, 16, 128), _z(4, 16, 64))}),
    (ValueError, {"cache": la.LatentCache(_z(4, 512), _z(4, 64))}),
    (ValueError, {"cache": la.LatentCache(_z(4, 16, 512), _z(4, 15, 64))}),
    (ValueError, {"cache": la.LatentCache(_z(4, 16, 512), _z(4, 16, 32))}),
    (TypeError, {"cache": la.LatentCache(_z(4, 16, 512), _z(4, 16, 64, dtype=torch.float32))}),
    (ValueError, {"cache": la.LatentCache(_z(4, 16, 512), _z(4, 16, 64), _z(4, 16, dtype=torch.float32))}),
    (ValueError, {"cache": la.LatentCache(_z(4, 16, 512).to(torch.float8_e4m3fn), _z(4, 16, 64).to(torch.float8_e4m3fn))}),
    (TypeError, {"cache": la.LatentCache(_z(4, 16, 512).to(torch.float8_e4m3fn), _z(4, 16, 64).to(torch.float8_e4m3fn),
                                         _z(4, 16))}),
    (ValueError, {"cache": la.LatentCache(_z(4, 16, 513)[..., 1:], _z(4, 16, 64))}),
    (ValueError, {"cache": la.LatentCache(_z(4, 512, 16).transpose(1, 2), _z(4, 16, 64))}),
    (RuntimeError, {"cache": la.LatentCache(_z(1, 16, 512).expand(4, 16, 512), _z(4, 16, 64))}),
    (RuntimeError, {"kv": _z(3, 576).requires_grad_()}),
    (ValueError, {}),  # host tensors
])
def test_append_refusals(error, change):
    with pytest.raises(error):
        la.latent_cache_append(**{**APPEND, "cache": _cache(), **change})


def test_append_without_key_part_refuses_odd_tables():
    for cols in (8, 24, 528):
        with pytest.raises(ValueError, match="multiple of 16"):
            la.latent_cache_append(_z(3, 512), _i(3), _i(3), _z(8, cols, dtype=torch.float32), _cache(P=0))


@pytest.mark.parametrize("error,weight", [(TypeError, _z(2, 16, 16, dtype=torch.float32)), (ValueError, _z(16, 16)),
                                          (ValueError, _z(2, 12, 16)), (ValueError, _z(2, 16, 12)),
                                          (ValueError, _z(0, 16, 16)), (RuntimeError, _z(2, 16, 16).requires_grad_()),
                                          (ValueError, _z(2, 16, 16))])
def test_prepare_head_projection_refusals(error, weight):
    with pytest.raises(error):
        la.prepare_head_projection(weight)


def test_head_projection_refusals():
    w = la.PreparedHeadProjection(torch.zeros((2, 1024), dtype=torch.int8), 2, 16, 16)
    for error, x, kw in ((TypeError, _z(3, 2, 16, dtype=torch.float32), {}), (ValueError, _z(3, 2, 17), {}),
                         (ValueError, _z(3, 1, 16), {}), (ValueError, _z(3, 2, 16), {"out": _z(3, 2, 15)}),
                         (TypeError, _z(3, 2, 16), {"out": _z(3, 2, 16, dtype=torch.float32)}),
                         (RuntimeError, _z(3, 2, 16).requires_grad_(), {}), (ValueError, _z(3, 2, 16), {})):
        with pytest.raises(error):
            la.head_projection(x, w, **kw)
    with pytest.raises(TypeError):
        la.head_projection(_z(3, 2, 16), _z(2, 16, 16))
    with pytest.raises(ValueError):
        la.head_projection(_z(3, 2, 16), la.PreparedHeadProjection(torch.zeros((2, 1000), dtype=torch.int8), 2, 16, 16))
    x = _z(3, 2, 16)
    with pytest.raises(RuntimeError):
        la.head_projection(x, w, out=x)


ABSORBED = dict(q_latent=_z(3, 4, 512), q_rope=_z(3, 4, 64), page_table=_i(3, 5), kv_lens=_i(3), scale=0.1)


@pytest.mark.parametrize("error,change", [
    (TypeError, {"q_latent": _z(3, 4, 512, dtype=torch.float32)}),
    (ValueError, {"q_latent": _z(3, 4, 256)}),
    (ValueError, {"q_latent": _z(3, 512)}),
    (ValueError, {"q_rope": None}),
    (ValueError, {"q_rope": _z(3, 4, 32)}),
    (ValueError, {"q_rope": _z(2, 4, 64)}),
    (TypeError, {"page_table": _i(3, 5, dtype=torch.int64)}),
    (ValueError, {"page_table": _i(3)}),
    (TypeError, {"kv_lens": _i(3, dtype=torch.int64)}),
    (ValueError, {"kv_lens": _i(2)}),
    (ValueError, {"page_table": _i(2, 5), "kv_lens": _i(2)}),
    (ValueError, {"query_starts": _i(3)}),
    (TypeError, {"query_starts": _i(4, dtype=torch.int64)}),
    (ValueError, {"scale": 0.0}),
    (ValueError, {"scale": -1.0}),
    (ValueError, {"scale": float("nan")}),
    (ValueError, {"scale": 1e-60}),
    (ValueError, {"out": _z(3, 4, 64)}),
    (RuntimeError, {"q_latent": _z(3, 4, 512).requires_grad_()}),
    (ValueError, {}),  # host tensors
])
def test_absorbed_refusals(error, change):
    with pytest.raises(error):
        la.absorbed_attention(**{**ABSORBED, "cache": _cache(), **change})


def test_absorbed_refuses_a_rope_part_without_a_cache_for_it():
    with pytest.raises(ValueError, match="q_rope"):
        la.absorbed_attention(**ABSORBED, cache=_cache(P=0))


EXPANDED = dict(q=_z(5, 4, 192), kv=_z(7, 4, 256), k_rope=_z(7, 64), query_starts=_i(3), scale=0.1)


@pytest.mark.parametrize("error,change", [
    (TypeError, {"q": _z(5, 4, 192, dtype=torch.float32)}),
    (TypeError, {"kv": _z(7, 4, 256, dtype=torch.float32)}),
    (TypeError, {"k_rope": _z(7, 64, dtype=torch.float32)}),
    (ValueError, {"q": _z(5, 192)}),
    (ValueError, {"q": _z(5, 4, 160)}),
    (ValueError, {"kv": _z(7, 3, 256)}),
    (ValueError, {"kv": _z(7, 4, 192)}),
    (ValueError, {"k_rope": _z(6, 64)}),
    (ValueError, {"k_rope": None}),
    (TypeError, {"query_starts": _i(3, dtype=torch.int64)}),
    (ValueError, {"query_starts": _i(0)}),
    (ValueError, {"kv_starts": _i(4)}),
    (ValueError, {"scale": float("inf")}),
    (ValueError, {"out": _z(5, 4, 192)}),
    (RuntimeError, {"kv": _z(7, 4, 256).requires_grad_()}),
    (ValueError, {}),  # host tensors
])
def test_expanded_refusals(error, change):
    with pytest.raises(error):
        la.expanded_attention(**{**EXPANDED, **change})


# ---- the C ABI -------------------------------------------------------------------------------------------------------


def _err(rc, code, text):
    assert rc == code, (rc, cabi.lib().fcmoe_last_error())
    assert text in cabi.lib().fcmoe_last_error(), cabi.lib().fcmoe_last_error()


def _desc(**kw):
    c = cabi.LatentCacheDesc(latent=4096, rope=4096, scale=None, pages=4, page_size=16, latent_dim=512, rope_dim=64,
                             latent_page_stride=16 * 512, latent_row_stride=512, rope_page_stride=16 * 64, rope_row_stride=64)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def test_cabi_refusals():
    L = cabi.lib()
    for fn in ("head_norm_rope", "latent_cache_append", "head_projection", "absorbed_attention", "expanded_attention"):
        _err(getattr(L, f"fcmoe_{fn}")(None, None), -1, b"NULL args")
    n = cabi.HeadNormRopeArgs(tokens=1, heads=1, dim=64, rope_dim=3)
    _err(L.fcmoe_head_norm_rope(n, None), -1, b"rope_dim")
    n.rope_dim = 64
    _err(L.fcmoe_head_norm_rope(n, None), -1, b"NULL pointer")
    n.tokens = 0
    assert L.fcmoe_head_norm_rope(n, None) == 0
    for bad in ({"latent_dim": 300}, {"rope_dim": 32}, {"page_size": 0}, {"latent": None}, {"rope": None}, {"e4m3": 1},
                {"latent_row_stride": 513}, {"rope_page_stride": 4}, {"latent": 4097}, {"pages": -1}):
        a = cabi.LatentAppendArgs(tokens=1, rot_dim=64, cache=_desc(**bad))
        assert L.fcmoe_latent_cache_append(a, None) == -1, bad
        b = cabi.AbsorbedArgs(tokens=1, heads=1, batch=1, scale=1.0, cache=_desc(**bad))
        assert L.fcmoe_absorbed_attention(b, None) == -1, bad
        assert L.fcmoe_absorbed_attention_workspace_bytes(b) == 0, bad
    a = cabi.LatentAppendArgs(tokens=1, rot_dim=32, cache=_desc())
    _err(L.fcmoe_latent_cache_append(a, None), -1, b"rotate")
    p = cabi.HeadProjectionArgs(tokens=1, heads=1, n=12, k=16)
    _err(L.fcmoe_head_projection(p, None), -1, b"multiples of 8")
    b = cabi.AbsorbedArgs(tokens=2, heads=1, batch=1, scale=1.0, cache=_desc())
    _err(L.fcmoe_absorbed_attention(b, None), -1, b"query_starts")
    b.batch, b.scale = 2, 0.0
    _err(L.fcmoe_absorbed_attention(b, None), -1, b"scale")
    b.scale, b.table_width = 1.0, 1
    _err(L.fcmoe_absorbed_attention(b, None), -1, b"NULL pointer")
    for k in ("q_latent", "q_rope", "kv_lens", "out", "page_table"):
        setattr(b, k, 4096)
    b.q_latent_token_stride = 513
    _err(L.fcmoe_absorbed_attention(b, None), -1, b"16 bytes")
    b.q_latent_token_stride = 512
    _err(L.fcmoe_absorbed_attention(b, None), -2, b"workspace")
    e = cabi.ExpandedArgs(tokens=1, keys=1, heads=1, batch=1, nope_dim=96, v_dim=96, scale=1.0)
    _err(L.fcmoe_expanded_attention(e, None), -1, b"128/128")
    e.nope_dim = e.v_dim = 128
    e.rope_dim = 64
    _err(L.fcmoe_expanded_attention(e, None), -1, b"NULL pointer")
    for k in ("q", "kv", "k_rope", "query_starts", "kv_starts", "out"):
        setattr(e, k, 4096)
    e.kv_token_stride = 1 << 24
    _err(L.fcmoe_expanded_attention(e, None), -1, b"2^24")
    e.kv_token_stride, e.keys = 256, 100000
    assert L.fcmoe_expanded_attention_workspace_bytes(e) > 0
    _err(L.fcmoe_expanded_attention(e, None), -2, b"workspace")


@pytest.mark.parametrize("mirror,name", [(cabi.HeadNormRopeArgs, "fcmoe_head_norm_rope_args"),
                                         (cabi.LatentCacheDesc, "fcmoe_latent_cache"),
                                         (cabi.LatentAppendArgs, "fcmoe_latent_append_args"),
                                         (cabi.HeadProjectionArgs, "fcmoe_head_projection_args"),
                                         (cabi.AbsorbedArgs, "fcmoe_absorbed_args"),
                                         (cabi.ExpandedArgs, "fcmoe_expanded_args")])
def test_ctypes_mirrors_the_header(tmp_path, mirror, name):
    src = tmp_path / "layout.c"
    lines = "".join(f'printf("{f} %zu\\n", offsetof({name}, {f}));' for f, _ in mirror._fields_)
    src.write_text(f'#include <stddef.h>\n#include <stdio.h>\n#include "fcmoe.h"\n'
                   f'int main(void) {{ {lines} printf("sizeof %zu\\n", sizeof({name})); return 0; }}\n')
    subprocess.run(["gcc", "-I", str(REPO / "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout
    got = dict((k, int(v)) for k, v in (line.split() for line in out.splitlines()))
    assert got.pop("sizeof") == ctypes.sizeof(mirror)
    assert got == {f: getattr(mirror, f).offset for f, _ in mirror._fields_}
