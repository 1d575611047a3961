"""Outputs that lie between the rows of a call's inputs, in one tensor with them."""

from __future__ import annotations

import pytest
import torch

from tests import latent_reference as ref
from tests.test_gpu_latent_attention import BF16, _expanded_inputs, _i32, _la, _Paged, _queries, _randn

pytestmark = pytest.mark.gpu


def test_outputs_between_the_inputs_rows(gpu):
    la = _la()
    table, pos = ref.rope_table(64, 50, "cuda"), torch.arange(11, device="cuda")
    buf = _randn(1, 11, 6, 400).to(BF16)
    x, out = buf[..., :192], buf[..., 200:392]
    want = la.head_norm_rope(x.contiguous(), pos, table)
    assert torch.equal(la.head_norm_rope(x, pos, table, out=out), want)
    odd, even = buf[:, 0::2, :192], buf[:, 1::2, :192]
    want = la.head_norm_rope(odd.contiguous(), pos, table, interleaved=False)
    assert torch.equal(la.head_norm_rope(odd, pos, table, interleaved=False, out=even), want)
    assert torch.equal(even, want)

    w = la.prepare_head_projection(_randn(2, 6, 128, 192).to(BF16))
    want = la.head_projection(odd.repeat(1, 2, 1), w)
    both = torch.cat([odd.repeat(1, 2, 1), torch.zeros((11, 6, 128), dtype=BF16, device="cuda")], -1)
    assert torch.equal(la.head_projection(both[..., :192], w, out=both[..., 192:]), want)
    assert torch.equal(both[..., :192], odd.repeat(1, 2, 1))


def test_attention_outputs_between_the_queries(gpu):
    la = _la()
    pg = _Paged(2, [70, 10, 300], 512, 64, BF16, page=16)
    ql, qr = _queries(7, 3, 16, 512, 64)
    want = la.absorbed_attention(ql, qr, pg.cache, pg.table, pg.lens, scale=0.07)
    buf = torch.cat([ql, qr, torch.zeros_like(ql)], -1)
    got = la.absorbed_attention(buf[..., :512], buf[..., 512:576], pg.cache, pg.table, pg.lens, scale=0.07, out=buf[..., 576:])
    assert torch.equal(got, want) and torch.equal(buf[..., :512], ql)
    q, kv, kr = _expanded_inputs(5, [70, 33], [70, 33], 4, 128, 64)
    want = la.expanded_attention(q, kv, kr, _i32([0, 70, 103]), scale=0.08)
    buf = torch.cat([q, torch.zeros((103, 4, 128), dtype=BF16, device="cuda")], -1)
    assert torch.equal(la.expanded_attention(buf[..., :192], kv, kr, _i32([0, 70, 103]), scale=0.08, out=buf[..., 192:]), want)
