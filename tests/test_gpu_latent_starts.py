"""Query starts of the latent attentions that are not in order: a start below an earlier one counts as that one, so
that no token belongs to two sequences and nothing is written outside the outputs and workspaces."""

from __future__ import annotations

import math

import pytest
import torch

from tests import latent_reference as ref
from tests.test_gpu_latent_attention import (BF16, E4M3, _check_absorbed, _expanded_inputs, _i32, _la, _Paged, _queries)

pytestmark = pytest.mark.gpu


def _followed(starts, tokens):
    out, high = [], 0
    for s in starts:
        high = max(high, min(max(s, 0), tokens))
        out.append(high)
    return out


def _outside(out, lse, starts):
    """Tokens before the first and behind the largest start."""
    for rows in (slice(0, starts[0]), slice(starts[-1], None)):
        assert bool((out[rows] == 0).all()) and bool((lse[rows] == -math.inf).all())


FALLING = [
    [0, 9, 0, 9, 0, 9, 0],        # every token named again and again
    [0, 3, 7, 0, 0, 0, 0],        # a batch padded with zeros
    [2, 5, 4, 8, 1, 6, 7],        # falls in the midst
    [4, -3, 20, 9, 2 ** 31 - 1, -2 ** 31, 5],
    [9, 8, 7, 6, 5, 4, 3],
]


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("H", [3, 16, 64, 128])
@pytest.mark.parametrize("starts", FALLING)
def test_absorbed_falling_starts(gpu, starts, H, dtype):
    lens = [70, 300, 5, 129, 64, 1]
    pg = _Paged(31, lens, 512, 64, dtype, page=16)
    ql, qr = _queries(31, 9, H, 512, 64)
    st = _followed(starts, 9)
    got = _la().absorbed_attention(ql, qr, pg.cache, pg.table, pg.lens, scale=0.07, query_starts=_i32(starts), return_lse=True)
    want, lse = _check_absorbed(pg, lens, ql, qr, st, 0.07)
    assert torch.equal(got[0], want) and torch.equal(got[1], lse)
    _outside(*got, st)


@pytest.mark.parametrize("H", [16, 128])
def test_absorbed_falling_starts_of_many_sequences(gpu, H):
    """Falls inside and between the groups of 64 sequences that a wave looks at."""
    g = torch.Generator().manual_seed(5)
    count, tokens = 200, 150
    starts = torch.randint(-5, tokens + 5, (count + 1,), generator=g).sort().values
    fall = torch.randint(0, count, (30,), generator=g)
    starts[fall] = torch.randint(0, tokens, (30,), generator=g)
    starts[64], starts[128] = 0, 3
    starts = starts.tolist()
    lens = [(53 * b) % 300 for b in range(count)]
    pg = _Paged(32, lens, 256, 64, BF16, page=32)
    ql, qr = _queries(32, tokens, H, 256, 64)
    st = _followed(starts, tokens)
    got = _la().absorbed_attention(ql, qr, pg.cache, pg.table, pg.lens, scale=0.07, query_starts=_i32(starts), return_lse=True)
    want, lse = _check_absorbed(pg, lens, ql, qr, st, 0.07)
    assert torch.equal(got[0], want) and torch.equal(got[1], lse)
    _outside(*got, st)


@pytest.mark.parametrize("tokens,batch", [(2, 32768), (1, 25000), (9, 64)])
def test_absorbed_falling_starts_stay_in_their_workspace(gpu, tokens, batch):
    """Far more sequences than tokens, each of which names all of them, through the C entry: what lies behind the
    workspace keeps its bytes."""
    import ctypes

    from fused_cpp_amd import cabi

    H, page, guard = 16, 64, 1 << 21
    pg = _Paged(33, [50], 512, 64, BF16, page=page, spare=0)
    ql, qr = _queries(33, tokens, H, 512, 64)
    ql, qr = ql.contiguous(), qr.contiguous()
    starts = _i32([0 if b % 2 == 0 else tokens for b in range(batch + 1)])
    lens, table = torch.full((batch,), 50, dtype=torch.int32, device="cuda"), pg.table[:, :1].expand(batch, 1).contiguous()
    out = torch.full((tokens, H, 512), 7.0, dtype=BF16, device="cuda")
    c = pg.cache
    a = cabi.AbsorbedArgs(q_latent=ql.data_ptr(), q_rope=qr.data_ptr(), tokens=tokens, heads=H, batch=batch,
                          q_latent_token_stride=H * 512, q_latent_head_stride=512, q_rope_token_stride=H * 64,
                          q_rope_head_stride=64, page_table=table.data_ptr(), table_width=1, page_table_stride=1,
                          kv_lens=lens.data_ptr(), query_starts=starts.data_ptr(), scale=0.07, out=out.data_ptr(),
                          out_token_stride=H * 512, out_head_stride=512, zero_uncovered=1)
    a.cache = cabi.LatentCacheDesc(latent=c.latent.data_ptr(), rope=c.rope.data_ptr(), pages=c.latent.shape[0], page_size=page,
                                   latent_dim=512, rope_dim=64, latent_page_stride=page * 512, latent_row_stride=512,
                                   rope_page_stride=page * 64, rope_row_stride=64)
    size = cabi.lib().fcmoe_absorbed_attention_workspace_bytes(ctypes.byref(a))
    assert size > 0
    ws = torch.full((size + guard,), 0x5A, dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = ws.data_ptr(), size
    assert cabi.lib().fcmoe_absorbed_attention(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert bool((ws[size:] == 0x5A).all())
    want, _, tol, _ = ref.absorbed(ql, qr, pg.rows, [50], [0, tokens], 0.07)
    ref.assert_within(out, want, tol)


@pytest.mark.parametrize("past", [0, 1500])
@pytest.mark.parametrize("starts", FALLING)
def test_expanded_falling_starts(gpu, starts, past):
    """Blocks of 128 rows, and of 256 (an average of more than 128 tokens and 1024 keys)."""
    by = 30 if past == 0 else 120
    tokens = 9 * by
    starts = [max(min(s, 100) * by, -2 ** 31) if abs(s) < 1000 else s for s in starts]
    lens = [40 + past, past, 300 + past, past, 77 + past, 5 + past]
    q, kv, kr = _expanded_inputs(34, [tokens], lens, 2, 128, 64)
    ks = [sum(lens[:b]) for b in range(7)]
    st = _followed(starts, tokens)
    got = _la().expanded_attention(q, kv, kr, _i32(starts), kv_starts=_i32(ks), scale=0.08, return_lse=True)
    want, wl, tol, ltol = ref.expanded(q, kv, kr, st, ks, 0.08, True)
    ref.assert_within(got[0], want, tol, "out")
    ref.assert_within(got[1], wl, ltol, "lse")
    _outside(*got, st)
