"""GPU selection of the positions that stay in a row whose columns and first tokens together pass 32 bits."""

from __future__ import annotations

import pytest
import torch

from tests import context_reference as cref
from tests.test_gpu_latent_attention import _i32
from tests.test_gpu_latent_context import _lc

pytestmark = pytest.mark.gpu


def test_heaviest_first_tokens_and_columns_past_32_bits(gpu):
    """2^30 + 2^17 columns of which 2^30 + 50 always stay: the slices of the last columns begin past 2^31."""
    S, sinks, recent, more = (1 << 30) + (1 << 17), (1 << 30) + 50, 70, 90
    keep = sinks + recent + more
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GiB of device memory")
    try:
        w = torch.zeros((1, S), device="cuda")
        g = torch.Generator(device="cuda").manual_seed(1)
        w[0, sinks:] = torch.rand(S - sinks, generator=g, device="cuda")
        positions, counts, kept = _lc().heaviest_positions(w, _i32([S]), keep, sinks=sinks, recent=recent)
        assert counts.tolist() == [keep]
        tail = cref.heaviest(w[0, sinks:].cpu().tolist(), S - sinks, more + recent, 0, recent)
        assert positions[0, sinks:].tolist() == [sinks + j for j in tail]
        assert torch.equal(kept[0, sinks:], w[0, sinks:][tail])
        assert torch.equal(positions[0, :sinks], torch.arange(sinks, dtype=torch.int32, device="cuda"))
        assert not bool(kept[0, :sinks].any())
    finally:
        w = positions = kept = None
        torch.cuda.empty_cache()
