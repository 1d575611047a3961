"""Outputs that share memory with what a call reads, or with themselves, are refused however both are strided; views
that only lie between one another's rows are not. Every check comes before the devices', so host tensors reach it: a
call that passes them ends with the refusal of the device."""

from __future__ import annotations

import random

import pytest
import torch

from fused_cpp_amd import latent_attention as la

BF16 = torch.bfloat16
TABLE = torch.zeros((8, 2))


def _z(*shape, dtype=BF16):
    return torch.zeros(shape, dtype=dtype)


def _i(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def _accepted(call):
    with pytest.raises(ValueError, match="device"):
        call()


def _refused(call):
    with pytest.raises(RuntimeError, match="overlap"):
        call()


def _norm(x, out, cos_sin=TABLE):
    return la.head_norm_rope(x, _i(x.shape[0]), cos_sin, out=out)


def test_norm_rope_views_of_one_buffer():
    buf = _z(3, 6, 16)
    _refused(lambda: _norm(buf[:, :4], buf[:, 1:5]))          # heads of one another's rows
    _refused(lambda: _norm(buf[..., :12], buf[..., 4:]))      # parts of one another's heads
    _refused(lambda: _norm(buf[:2], buf[1:]))
    _refused(lambda: _norm(buf[:, :4, :8], buf[:, :4, 7:15]))
    _refused(lambda: _norm(buf.flip(0)[:, :4, :8].contiguous(), buf[:, :4, :1].expand(3, 4, 8)))
    _refused(lambda: _norm(buf[:, :3, :8], buf.as_strided((3, 3, 8), (8, 4, 1))))  # an output over itself
    _accepted(lambda: _norm(buf, buf))
    _accepted(lambda: _norm(buf[:, 1:3, 4:12], buf[:, 1:3, 4:12]))
    _accepted(lambda: _norm(buf[:, :3], buf[:, 3:]))
    _accepted(lambda: _norm(buf[..., :8], buf[..., 8:]))
    _accepted(lambda: _norm(buf[:, 0::2], buf[:, 1::2]))
    _accepted(lambda: _norm(buf[..., 0::2], buf[..., 1::2]))
    _accepted(lambda: _norm(buf[:, :1], buf[:, 1:2]))
    one = _z(1, 3, 8)
    _accepted(lambda: _norm(one, one.as_strided((1, 3, 8), (77, 8, 1))))  # the stride of a single token is not used


def test_norm_rope_other_inputs():
    raw = torch.zeros(4096, dtype=torch.uint8)
    x, out = _z(3, 2, 8), raw[:96].view(BF16).view(3, 2, 8)
    _refused(lambda: _norm(x, out, raw[64:128].view(torch.float32).view(8, 2)))
    _accepted(lambda: _norm(x, out, raw[96:160].view(torch.float32).view(8, 2)))
    _refused(lambda: la.head_norm_rope(x, raw[88:100].view(torch.int32), TABLE, out=out))
    _refused(lambda: la.head_norm_rope(x, _i(3), TABLE, weight=raw[:16].view(BF16), out=out))


def _places(t):
    at = torch.zeros(t.shape, dtype=torch.int64)
    for d in range(t.dim()):
        at += (torch.arange(t.shape[d]) * t.stride(d)).view([-1 if e == d else 1 for e in range(t.dim())])
    return (at + t.storage_offset()).flatten().tolist()


def test_against_every_place():
    """Random strided views of a small buffer: refused exactly where two places are one."""
    rng = random.Random(7)
    buf = _z(400)
    seen = [0, 0]
    for _ in range(3000):
        shape = (rng.randint(1, 4), rng.randint(1, 3), rng.randint(2, 5))
        views = []
        for _ in range(2):
            kind = rng.random()
            if kind < 0.4:  # dimensions inside one another, in any order
                order, stride, span = rng.sample(range(3), 3), [0, 0, 0], 1
                for d in order:
                    stride[d] = span + rng.randint(0, 2)
                    span = stride[d] * shape[d]
            else:
                stride = [rng.randint(1, 24) for _ in range(3)]
            if views and kind < 0.3:
                stride = list(views[0].stride())
            most = sum((n - 1) * s for n, s in zip(shape, stride))
            if most >= 399:
                break
            views.append(buf.as_strided(shape, stride, rng.randint(0, min(399 - most, 60))))
        if len(views) < 2:
            continue
        x, out = views
        px, po = _places(x), _places(out)
        same = px == po and all(n == 1 or a == b for n, a, b in zip(shape, x.stride(), out.stride()))
        shares = len(set(po)) < len(po) or (not same and bool(set(px) & set(po)))
        seen[shares] += 1
        (_refused if shares else _accepted)(lambda: _norm(x, out))
    assert min(seen) > 300, seen


def test_large_views_of_one_buffer():
    """Layouts of real size are told apart without looking at every place."""
    buf = _z(4096, 16, 192)
    _accepted(lambda: _norm(buf[..., :96], buf[..., 96:]))
    _refused(lambda: _norm(buf[..., :97], buf[..., 95:]))
    _accepted(lambda: _norm(buf[:2048], buf[2048:]))
    _refused(lambda: _norm(buf[:2049], buf[2047:]))
    _accepted(lambda: _norm(buf.view(16, 4096, 192).transpose(0, 1)[..., :96], buf.view(16, 4096, 192).transpose(0, 1)[..., 96:]))


def test_head_projection():
    w = la.PreparedHeadProjection(torch.zeros((2, 1024), dtype=torch.int8), 2, 16, 16)
    buf = _z(3, 4, 32)
    _refused(lambda: la.head_projection(buf[:, :2, :16], w, out=buf[:, 1:3, :16]))
    _refused(lambda: la.head_projection(buf[:, :2, :16], w, out=buf[:, :2, 15:31]))
    _accepted(lambda: la.head_projection(buf[:, :2, :16], w, out=buf[:, :2, 16:]))
    _refused(lambda: la.head_projection(_z(3, 2, 16), w, out=w.packed.view(-1)[:192].view(BF16).view(3, 2, 16)))


def _absorbed(**change):
    c = la.allocate_latent_cache(4, 16, device="cpu")
    kw = dict(q_latent=_z(3, 4, 512), q_rope=_z(3, 4, 64), cache=c, page_table=_i(3, 5), kv_lens=_i(3), scale=0.1)
    return lambda: la.absorbed_attention(**{**kw, **change})


def test_absorbed():
    q = _z(3, 8, 1088)
    _accepted(_absorbed(q_latent=q[:, :4, :512], q_rope=q[:, :4, 512:576], out=q[:, :4, 576:]))
    _refused(_absorbed(q_latent=q[:, :4, :512], out=q[:, 1:5, :512]))
    _refused(_absorbed(q_latent=q[:, :4, :512], q_rope=q[:, :4, 512:576], out=q[:, :4, 575:1087]))
    c = la.allocate_latent_cache(4, 16, device="cpu")
    _refused(_absorbed(cache=c, out=c.latent.view(-1)[:3 * 4 * 512].view(3, 4, 512)))
    c8 = la.allocate_latent_cache(4, 16, dtype=torch.float8_e4m3fn, device="cpu")
    _refused(_absorbed(cache=c8, out=c8.latent.view(-1)[:3 * 4 * 1024].view(BF16).view(3, 4, 512)))
    out = _z(3, 4, 512)
    _refused(_absorbed(out=out, kv_lens=out.view(-1).view(torch.int32)[-3:]))
    _refused(_absorbed(out=out, page_table=out.view(-1).view(torch.int32)[:15].view(3, 5)))


def test_expanded():
    kw = dict(kv=_z(7, 4, 256), k_rope=_z(7, 64), query_starts=_i(3), scale=0.1)
    q = _z(5, 6, 320)
    _accepted(lambda: la.expanded_attention(q[:, :4, :192], **kw, out=q[:, :4, 192:]))
    _refused(lambda: la.expanded_attention(q[:, :4, :192], **kw, out=q[:, 1:5, :128]))
    both = _z(7, 5, 256)
    _refused(lambda: la.expanded_attention(q[:, :4, :192], **{**kw, "kv": both[:, :4]}, out=both[:5, 1:5, 64:192]))
    _accepted(lambda: la.expanded_attention(q[:, :2, :192], **{**kw, "kv": both[:, :2]}, out=both[:5, 2:4, 64:192]))


def test_append():
    both = _z(4, 16, 576)
    kv, slots, table = _z(3, 576), _i(3), torch.zeros((8, 64))
    call = lambda c, kv=kv: lambda: la.latent_cache_append(kv, _i(3), slots, table, c)  # noqa: E731
    _accepted(call(la.LatentCache(both[..., :512], both[..., 512:])))
    _refused(call(la.LatentCache(both[..., :512], both[..., 504:568])))
    _refused(call(la.LatentCache(both[..., :512], both[..., 512:]), both[0, :3]))
    _refused(call(la.LatentCache(both.as_strided((4, 16, 512), (512, 512, 1)), _z(4, 16, 64))))
    raw = torch.zeros(256, dtype=torch.uint8)
    c8 = la.LatentCache(torch.zeros((4, 16, 512), dtype=torch.uint8).view(torch.float8_e4m3fn),
                        torch.zeros((4, 16, 64), dtype=torch.uint8).view(torch.float8_e4m3fn),
                        raw.view(torch.float32).view(4, 16))
    _accepted(call(c8))
    _refused(call(la.LatentCache(c8.latent, c8.rope, c8.latent.view(torch.uint8).view(-1)[:256].view(torch.float32).view(4, 16))))
