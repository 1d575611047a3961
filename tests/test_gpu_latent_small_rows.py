"""8-bit rows whose values are too small for a scale of their own."""

from __future__ import annotations

import pytest
import torch

from tests import latent_reference as ref
from tests.test_gpu_latent_attention import BF16, E4M3, _cache, _cache_rows, _la

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("P", [64, 0])
def test_append_rows_below_a_scale(gpu, P):
    """Largest values around 448 times the smallest binary32 number: max / 448 is some of its steps, one, or 0. With 0
    there is no scale to divide by; the row is stored as zeros, the zeros in it among them."""
    la = _la()
    smallest = 2.0 ** -133  # of bf16; a normalised value of 2^-k times it is 2^(16 - k) steps of 2^-149
    c = _cache(1, 8, 512, P, E4M3)
    kv = torch.zeros((6, 512 + P), dtype=BF16, device="cuda")
    w = torch.full((512,), smallest, dtype=BF16, device="cuda")
    for t, k in enumerate((0, 4, 7, 9, 12, 40)):
        kv[t, 1:512:3] = 2.0 ** -k
    pos = torch.arange(6, device="cuda")
    table = ref.rope_table(P or 64, 8, "cuda")[:, :P or 64] * 0 + torch.cat([torch.ones((P or 64) // 2), torch.zeros((P or 64) // 2)]).cuda()
    la.latent_cache_append(kv, pos, pos, table, c, weight=w, eps=1.0)  # with eps 1 a row of 2^-k keeps about that size
    x = kv.to(ref.F64)
    want = torch.cat([ref.norm(x[:, :512], w, 1.0), x[:, 512:]], 1)
    got = _cache_rows(c, pos)
    assert bool(torch.isfinite(got).all()) and bool((got[want == 0] == 0).all())
    # a value rounds to binary32's steps, its scale too (by at most half a step, 448 of which a value can be off by),
    # then to e4m3
    step = 2.0 ** -149
    ref.assert_within(got, want, 2.0 ** -4 * want.abs() + 2.0 ** -10 * c.scale.view(-1)[pos].to(ref.F64)[:, None] * (
        c.scale.view(-1)[pos].to(ref.F64)[:, None] < 1) + 450 * step)
    assert bool((c.scale.view(-1)[pos] > 0).all())
