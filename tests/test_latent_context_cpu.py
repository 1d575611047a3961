"""Attention over parts of a latent context without a GPU: refusals (reached with host tensors, devices are checked
last), the C ABI's argument checks, and the ctypes mirror of its structures."""

from __future__ import annotations

import ctypes
import subprocess

import pytest
import torch
import torch.autograd.forward_ad as fwd

from fused_cpp_amd import cabi
from fused_cpp_amd import latent_attention as la
from fused_cpp_amd import latent_context as lc
from tests import context_reference as cref
from tests.test_latent_attention_cpu import REPO, _cache, _desc, _err, _i, _z

F32 = torch.float32
CACHE = _cache()
ABSORBED = dict(q_latent=_z(3, 4, 512), q_rope=_z(3, 4, 64), cache=CACHE, page_table=_i(3, 5), kv_lens=_i(3), scale=0.1)
EXPANDED = dict(q=_z(5, 4, 192), kv=_z(7, 4, 256), k_rope=_z(7, 64), query_starts=_i(3), scale=0.1)


def _tree(masks=None, depths=None):
    return lc.DraftTree(_i(3, 2, dtype=torch.int64) if masks is None else masks, _i(3) if depths is None else depths)


def test_public_names():
    import fused_cpp_amd

    assert "latent_context" in fused_cpp_amd.__all__
    assert set(lc.__all__) == {"DraftTree", "attention_weights", "draft_tree", "heaviest_positions", "latent_cache_move"}


@pytest.mark.parametrize("error,change", [
    (ValueError, {"window": 0}),
    (ValueError, {"window": -3}),
    (ValueError, {"sinks": 4}),
    (ValueError, {"window": 8, "sinks": -1}),
    (TypeError, {"window": 8.5}),
    (TypeError, {"tree": _i(3, 1, dtype=torch.int64), "query_starts": _i(4)}),
    (ValueError, {"tree": _tree()}),
    (TypeError, {"tree": _tree(masks=_i(3, 2)), "query_starts": _i(4)}),
    (ValueError, {"tree": _tree(masks=_i(4, 2, dtype=torch.int64)), "query_starts": _i(4)}),
    (ValueError, {"tree": _tree(masks=_i(3, 0, dtype=torch.int64)), "query_starts": _i(4)}),
    (ValueError, {"tree": _tree(masks=_i(3, 17, dtype=torch.int64)), "query_starts": _i(4)}),
    (ValueError, {"tree": _tree(masks=_i(3, dtype=torch.int64)), "query_starts": _i(4)}),
    (TypeError, {"tree": _tree(depths=_i(3, dtype=torch.int64)), "query_starts": _i(4)}),
    (ValueError, {"tree": _tree(depths=_i(2)), "query_starts": _i(4)}),
    (ValueError, {"window": 8, "sinks": 2, "tree": _tree(), "query_starts": _i(4)}),  # host tensors
])
def test_absorbed_refusals(error, change):
    with pytest.raises(error):
        la.absorbed_attention(**{**ABSORBED, **change})


@pytest.mark.parametrize("error,change", [
    (ValueError, {"window": 0}),
    (ValueError, {"sinks": 1}),
    (ValueError, {"window": 5, "sinks": -1}),
    (ValueError, {"window": 5, "causal": False}),
    (ValueError, {"window": 5}),  # host tensors
])
def test_expanded_refusals(error, change):
    with pytest.raises(error):
        la.expanded_attention(**{**EXPANDED, **change})


def test_absorbed_out_may_not_lie_on_the_masks():
    both = torch.zeros(3 * 4 * 512 * 2, dtype=torch.uint8)
    out = both.view(torch.bfloat16).view(3, 4, 512)
    masks = both.view(torch.int64)[:6].view(3, 2)
    with pytest.raises(RuntimeError, match="overlap"):
        la.absorbed_attention(**ABSORBED, tree=_tree(masks=masks), query_starts=_i(4), out=out)


@pytest.mark.parametrize("error,change", [
    (TypeError, {"parents": _i(5, dtype=torch.int64)}),
    (ValueError, {"parents": _i(5, 1)}),
    (TypeError, {"query_starts": _i(3, dtype=torch.int64)}),
    (ValueError, {"query_starts": _i(0)}),
    (ValueError, {"query_starts": _i(3, 1)}),
    (ValueError, {"max_nodes": 0}),
    (ValueError, {"max_nodes": 1025}),
    (ValueError, {}),  # host tensors
])
def test_draft_tree_refusals(error, change):
    with pytest.raises(error):
        lc.draft_tree(**{**dict(parents=_i(5), query_starts=_i(3), max_nodes=5), **change})


WEIGHTS = dict(q_latent=_z(3, 4, 512), q_rope=_z(3, 4, 64), cache=CACHE, page_table=_i(3, 5), kv_lens=_i(3),
               lse=_z(3, 4, dtype=F32), scale=0.1, previous=_z(3, 80, dtype=F32))


@pytest.mark.parametrize("error,change", [
    (TypeError, {"q_latent": _z(3, 4, 512, dtype=F32)}),
    (ValueError, {"q_latent": _z(3, 4, 256)}),
    (ValueError, {"q_latent": _z(3, 0, 512)}),
    (ValueError, {"q_rope": None}),
    (ValueError, {"q_rope": _z(3, 5, 64)}),
    (TypeError, {"page_table": _i(3, 5, dtype=torch.int64)}),
    (ValueError, {"page_table": _i(3)}),
    (TypeError, {"kv_lens": _i(3, dtype=torch.int64)}),
    (ValueError, {"kv_lens": _i(4)}),
    (ValueError, {"page_table": _i(2, 5), "kv_lens": _i(2)}),
    (TypeError, {"lse": _z(3, 4)}),
    (ValueError, {"lse": _z(3, 5, dtype=F32)}),
    (TypeError, {"query_starts": _i(4, dtype=torch.int64)}),
    (ValueError, {"query_starts": _i(3)}),
    (TypeError, {"previous": _z(3, 80)}),
    (ValueError, {"previous": _z(2, 80, dtype=F32)}),
    (TypeError, {"out": _z(3, 80)}),
    (ValueError, {"out": _z(3, 81, dtype=F32)}),
    (ValueError, {"out": _z(80, 3, dtype=F32).T}),
    (RuntimeError, {"out": _z(3, 80, dtype=F32).requires_grad_()}),
    (RuntimeError, {"out": _z(1, 80, dtype=F32).expand(3, 80)}),
    (ValueError, {"scale": 0.0}),
    (ValueError, {"scale": float("nan")}),
    (ValueError, {"scale": 1e-60}),
    (ValueError, {}),  # host tensors
])
def test_weights_refusals(error, change):
    with pytest.raises(error):
        lc.attention_weights(**{**WEIGHTS, **change})


def test_weights_in_place_or_apart():
    both = _z(4, 80, dtype=F32)
    with pytest.raises(RuntimeError, match="overlap"):
        lc.attention_weights(**{**WEIGHTS, "previous": both[:3], "out": both[1:]})
    with pytest.raises(ValueError, match="device"):
        lc.attention_weights(**{**WEIGHTS, "previous": both[:3], "out": both[:3]})
    lse = _z(3, 80, dtype=F32)
    with pytest.raises(RuntimeError, match="overlap"):
        lc.attention_weights(**{**WEIGHTS, "lse": lse[:, :4], "out": lse})


HEAVY = dict(weights=_z(3, 80, dtype=F32), kv_lens=_i(3), keep=8, sinks=2, recent=3)


@pytest.mark.parametrize("error,change", [
    (TypeError, {"weights": _z(3, 80)}),
    (ValueError, {"weights": _z(80, dtype=F32)}),
    (TypeError, {"kv_lens": _i(3, dtype=torch.int64)}),
    (ValueError, {"kv_lens": _i(2)}),
    (ValueError, {"keep": 0}),
    (ValueError, {"keep": 1 << 40}),
    (ValueError, {"sinks": -1}),
    (ValueError, {"recent": -1}),
    (ValueError, {"sinks": 6, "recent": 3}),
    (ValueError, {"sinks": 9, "recent": 0}),
    (ValueError, {"sinks": (1 << 63) - 1, "recent": 1}),
    (RuntimeError, {"weights": _z(3, 80, dtype=F32).requires_grad_()}),
    (ValueError, {}),  # host tensors
])
def test_heaviest_refusals(error, change):
    kw = {**HEAVY, **change}
    with pytest.raises(error):
        lc.heaviest_positions(kw["weights"], kw["kv_lens"], kw["keep"], sinks=kw["sinks"], recent=kw["recent"])


MOVE = dict(cache=CACHE, page_table=_i(3, 5), positions=_i(3, 4), counts=_i(3), starts=_i(3), to_table=_i(3, 2))


@pytest.mark.parametrize("error,change", [
    (TypeError, {"page_table": _i(3, 5, dtype=torch.int64)}),
    (ValueError, {"page_table": _i(15)}),
    (TypeError, {"positions": _i(3, 4, dtype=torch.int64)}),
    (ValueError, {"positions": _i(2, 4)}),
    (ValueError, {"positions": _i(3)}),
    (TypeError, {"counts": _i(3, dtype=torch.int64)}),
    (ValueError, {"counts": _i(4)}),
    (TypeError, {"starts": _i(3, dtype=torch.int64)}),
    (ValueError, {"starts": _i(2)}),
    (TypeError, {"to_table": _i(3, 2, dtype=torch.int64)}),
    (ValueError, {"to_table": _i(2, 2)}),
    (TypeError, {"cache": la.LatentCache(_z(4, 16, 512, dtype=torch.float16), _z(4, 16, 64, dtype=torch.float16))}),
    (RuntimeError, {"cache": la.LatentCache(_z(4, 16, 512).requires_grad_(), _z(4, 16, 64))}),
    (RuntimeError, {"cache": la.LatentCache(_z(1, 16, 512).expand(4, 16, 512), _z(4, 16, 64))}),
    (ValueError, {}),  # host tensors
])
def test_move_refusals(error, change):
    with pytest.raises(error):
        lc.latent_cache_move(**{**MOVE, **change})


def test_move_cache_apart_from_what_is_read():
    raw = torch.zeros(4 * 16 * 512 * 2, dtype=torch.uint8)
    cache = la.LatentCache(raw.view(torch.bfloat16).view(4, 16, 512), _z(4, 16, 64))
    with pytest.raises(RuntimeError, match="overlap"):
        lc.latent_cache_move(**{**MOVE, "cache": cache, "counts": raw.view(torch.int32)[:3]})


CALLS = {
    "absorbed_attention": (la.absorbed_attention, {**ABSORBED, "window": 4}),
    "expanded_attention": (la.expanded_attention, {**EXPANDED, "window": 4}),
    "attention_weights": (lc.attention_weights, {**WEIGHTS, "out": _z(3, 80, dtype=F32)}),
    "heaviest_positions": (lc.heaviest_positions, HEAVY),
}


@pytest.mark.parametrize("name,arg", [(name, arg) for name, (_, kw) in CALLS.items() for arg, v in kw.items()
                                      if isinstance(v, torch.Tensor) and v.is_floating_point()])
def test_tangents_are_refused(name, arg):
    fn, kw = CALLS[name]
    with fwd.dual_level():
        dual = fwd.make_dual(kw[arg], torch.ones_like(kw[arg]))
        with pytest.raises(RuntimeError, match="tangent"):
            fn(**{**kw, arg: dual})


def test_cache_tangents_are_refused():
    with fwd.dual_level():
        cache = la.LatentCache(fwd.make_dual(CACHE.latent, torch.ones_like(CACHE.latent)), CACHE.rope)
        with pytest.raises(RuntimeError, match="tangent"):
            lc.attention_weights(**{**WEIGHTS, "cache": cache})
        with pytest.raises(RuntimeError, match="tangent"):
            lc.latent_cache_move(**{**MOVE, "cache": cache})


# ---- the C ABI -------------------------------------------------------------------------------------------------------


def test_cabi_masked_refusals():
    L = cabi.lib()
    b = cabi.AbsorbedArgs(tokens=2, heads=1, batch=2, scale=1.0, cache=_desc(), table_width=1)
    m = cabi.KeyMask(window=5, sinks=2)
    _err(L.fcmoe_absorbed_attention_masked(b, None, None), -1, b"NULL mask")
    _err(L.fcmoe_absorbed_attention_masked(None, m, None), -1, b"NULL args")
    assert L.fcmoe_absorbed_attention_masked_workspace_bytes(b, m) > 0
    for bad in ({"window": -1}, {"sinks": -1}, {"tree_masks": 4096, "mask_words": 1},
                {"tree_masks": 4096, "tree_depths": 4096, "mask_words": 17},
                {"tree_masks": 4100, "tree_depths": 4096, "mask_words": 1},
                {"tree_masks": 4096, "tree_depths": 4096, "mask_words": 1, "mask_stride": 1 << 40}):
        c = cabi.AbsorbedArgs(tokens=2, heads=1, batch=2, scale=1.0, cache=_desc(), table_width=1, query_starts=4096)
        assert L.fcmoe_absorbed_attention_masked(c, cabi.KeyMask(**bad), None) == -1, bad
        assert L.fcmoe_absorbed_attention_masked_workspace_bytes(c, cabi.KeyMask(**bad)) == 0, bad
    t = cabi.KeyMask(tree_masks=4096, tree_depths=4096, mask_words=1, mask_stride=1)
    _err(L.fcmoe_absorbed_attention_masked(b, t, None), -1, b"query_starts")
    for k in ("q_latent", "q_rope", "kv_lens", "out", "page_table"):
        setattr(b, k, 4096)
    _err(L.fcmoe_absorbed_attention_masked(b, m, None), -2, b"workspace")
    e = cabi.ExpandedArgs(tokens=1, keys=100000, heads=1, batch=1, nope_dim=128, v_dim=128, rope_dim=64, scale=1.0, causal=1)
    _err(L.fcmoe_expanded_attention_masked(e, None, None), -1, b"NULL")
    _err(L.fcmoe_expanded_attention_masked(e, cabi.KeyMask(window=-2), None), -1, b"negative")
    _err(L.fcmoe_expanded_attention_masked(e, t, None), -1, b"absorbed")
    e.causal = 0
    _err(L.fcmoe_expanded_attention_masked(e, m, None), -1, b"causal")
    e.causal = 1
    for k in ("q", "kv", "k_rope", "query_starts", "kv_starts", "out"):
        setattr(e, k, 4096)
    assert L.fcmoe_expanded_attention_masked_workspace_bytes(e, cabi.KeyMask(window=9000)) > 0
    _err(L.fcmoe_expanded_attention_masked(e, cabi.KeyMask(window=9000), None), -2, b"workspace")


def test_cabi_windows_past_32_bits_plan_as_ones_past_the_context():
    L = cabi.lib()
    b = cabi.AbsorbedArgs(tokens=2, heads=16, batch=2, scale=1.0, cache=_desc(), table_width=1 << 12)
    e = cabi.ExpandedArgs(tokens=1, keys=100000, heads=1, batch=1, nope_dim=128, v_dim=128, rope_dim=64, scale=1.0, causal=1)
    wide = cabi.KeyMask(window=1 << 30, sinks=1 << 30)
    for window, sinks in ((1 << 62, 1 << 62), ((1 << 63) - 1, 0), ((1 << 63) - 1, (1 << 63) - 1), (5, (1 << 63) - 1)):
        m = cabi.KeyMask(window=window, sinks=sinks)
        for fn, args in ((L.fcmoe_absorbed_attention_masked_workspace_bytes, b), (L.fcmoe_expanded_attention_masked_workspace_bytes, e)):
            assert fn(args, m) == fn(args, wide) > 0, (window, sinks)


def test_cabi_refusals():
    L = cabi.lib()
    for fn in ("attention_weights", "latent_cache_move"):
        _err(getattr(L, f"fcmoe_{fn}")(None, None), -1, b"NULL args")
    _err(L.fcmoe_draft_tree(None, 3, None, 1, 1, None, None, None), -1, b"NULL pointer")
    assert L.fcmoe_draft_tree(None, 0, None, 1, 1, None, None, None) == 0
    for tokens, batch, words in ((-1, 1, 1), (1, 0, 1), (1, 1, 0), (1, 1, 17), (1 << 40, 1, 1)):
        _err(L.fcmoe_draft_tree(4096, tokens, 4096, batch, words, 4096, 4096, None), -1, b"bad shape")
    heavy = lambda **kw: [{**dict(w=4096, batch=2, positions=9, stride=9, lens=4096, keep=4, sinks=1, recent=1, o=4096, c=4096,  # noqa: E731
                                  k=4096, ws=None, nb=0, s=None), **kw}[n]
                         for n in ("w", "batch", "positions", "stride", "lens", "keep", "sinks", "recent", "o", "c", "k", "ws", "nb", "s")]
    for bad in ({"keep": 0}, {"sinks": -1}, {"recent": -1}, {"sinks": 4}, {"positions": -1}, {"positions": 1 << 40}, {"batch": -1}):
        _err(L.fcmoe_heaviest_positions(*heavy(**bad)), -1, b"bad shape")
    _err(L.fcmoe_heaviest_positions(*heavy(w=None)), -1, b"NULL pointer")
    assert L.fcmoe_heaviest_positions(*heavy(batch=0)) == 0
    assert L.fcmoe_heaviest_positions_workspace_bytes(2, 8192, 4, 1, 1) == 0
    need = L.fcmoe_heaviest_positions_workspace_bytes(2, 8193, 4, 1, 1)
    assert need > 2 * 2 * 8192 * 4
    _err(L.fcmoe_heaviest_positions(*heavy(positions=8193, ws=4096, nb=need - 1)), -2, b"workspace")
    _err(L.fcmoe_heaviest_positions(*heavy(positions=8193, ws=4100, nb=need)), -1, b"unaligned")
    w = cabi.AttentionWeightsArgs(tokens=2, heads=1, batch=1, scale=1.0, cache=_desc())
    _err(L.fcmoe_attention_weights(w, None), -1, b"query_starts")
    w.batch, w.scale, w.positions = 2, -1.0, 10
    _err(L.fcmoe_attention_weights(w, None), -1, b"scale")
    w.scale = 1.0
    _err(L.fcmoe_attention_weights(w, None), -1, b"NULL pointer")
    w.positions = 0
    assert L.fcmoe_attention_weights(w, None) == 0
    w.positions, w.heads, w.table_width = 4000, 1000, 100
    for k in ("q_latent", "q_rope", "kv_lens", "out", "page_table", "lse"):
        setattr(w, k, 4096)
    w.q_rope_head_stride = 60
    _err(L.fcmoe_attention_weights(w, None), -1, b"16 bytes")
    w.q_rope_head_stride = 64
    assert L.fcmoe_attention_weights_workspace_bytes(w) > 0
    _err(L.fcmoe_attention_weights(w, None), -2, b"workspace")
    m = cabi.LatentMoveArgs(cache=_desc(), batch=1, most=4, table_width=2)
    _err(L.fcmoe_latent_cache_move(m, None), -1, b"NULL pointer")
    m.most = -1
    _err(L.fcmoe_latent_cache_move(m, None), -1, b"bad shape")
    m.most = 0
    assert L.fcmoe_latent_cache_move(m, None) == 0
    m.cache = _desc(page_size=0)
    assert L.fcmoe_latent_cache_move(m, None) == -1


@pytest.mark.parametrize("tokens,heads", [(1 << 60, 16), (1 << 62, 4), ((1 << 63) - 1, 1), (1 << 31, 1)])
def test_cabi_token_counts_past_the_products(tokens, heads):
    L = cabi.lib()
    a = cabi.AbsorbedArgs(tokens=tokens, heads=heads, batch=1, scale=1.0, cache=_desc(), table_width=1, query_starts=4096,
                          q_latent=4096, q_rope=4096, kv_lens=4096, out=4096, page_table=4096)
    m = cabi.KeyMask(tree_masks=4096, tree_depths=4096, mask_words=1, mask_stride=1, window=4)
    assert L.fcmoe_absorbed_attention_masked_workspace_bytes(a, m) == 0
    assert L.fcmoe_absorbed_attention_masked(a, m, None) == -1
    w = cabi.AttentionWeightsArgs(tokens=tokens, heads=heads, batch=1, scale=1.0, cache=_desc(), table_width=1, query_starts=4096,
                                  q_latent=4096, q_rope=4096, kv_lens=4096, out=4096, page_table=4096, lse=4096, positions=9)
    assert L.fcmoe_attention_weights_workspace_bytes(w) == 0
    assert L.fcmoe_attention_weights(w, None) == -1
    e = cabi.ExpandedArgs(tokens=tokens, keys=1, heads=heads, batch=1, nope_dim=128, v_dim=128, scale=1.0, causal=1)
    assert L.fcmoe_expanded_attention_masked(e, cabi.KeyMask(window=4), None) == -1


@pytest.mark.parametrize("mirror,name", [(cabi.KeyMask, "fcmoe_key_mask"),
                                         (cabi.AttentionWeightsArgs, "fcmoe_attention_weights_args"),
                                         (cabi.LatentMoveArgs, "fcmoe_latent_move_args")])
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


# ---- the reference itself ---------------------------------------------------------------------------------------------


def test_reference_windows_and_trees():
    k = cref.seen_by_window(2, 6, 3, 1, "cpu")
    assert k.int().tolist() == [[1, 0, 1, 1, 1, 0], [1, 0, 0, 1, 1, 1]]
    t = cref.seen_by_tree([-1, 0, 0, 1], 6, device="cpu")
    assert t.int().tolist() == [[1, 1, 1, 0, 0, 0], [1, 1, 1, 1, 0, 0], [1, 1, 1, 0, 1, 0], [1, 1, 1, 1, 0, 1]]
    t = cref.seen_by_tree([-1, 0, 1], 6, window=2, sinks=1, device="cpu")
    assert t.int().tolist() == [[1, 0, 1, 1, 0, 0], [1, 0, 0, 1, 1, 0], [1, 0, 0, 1, 1, 1]]
    assert cref.heaviest([1.0, 5.0, 5.0, 0.0, 5.0, 2.0], 6, 3, 1, 1) == [0, 1, 5]
    assert cref.heaviest([1.0, 5.0], 6, 3, 1, 1) == [0, 1]
