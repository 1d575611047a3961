"""Token counts whose products pass 64 bits are refused at the C entries, before anything is sized or launched by them."""

from __future__ import annotations

import pytest

from fused_cpp_amd import cabi


@pytest.mark.parametrize("tokens,heads", [(1 << 60, 16), (1 << 62, 4), ((1 << 63) - 1, 1), (1 << 31, 1)])
def test_token_counts_past_the_products(tokens, heads):
    lib = cabi.lib()
    cache = cabi.LatentCacheDesc(latent=4096, rope=4096, pages=4, page_size=64, latent_dim=512, rope_dim=64,
                                 latent_page_stride=64 * 512, latent_row_stride=512, rope_page_stride=64 * 64, rope_row_stride=64)
    a = cabi.AbsorbedArgs(tokens=tokens, heads=heads, batch=1, scale=1.0, cache=cache, table_width=1, query_starts=4096,
                          q_latent=4096, q_rope=4096, kv_lens=4096, out=4096, page_table=4096)
    assert lib.fcmoe_absorbed_attention_workspace_bytes(a) == 0
    assert lib.fcmoe_absorbed_attention(a, None) == -1
    n = cabi.HeadNormRopeArgs(tokens=tokens, heads=heads, dim=64, x=4096, out=4096, positions=4096)
    assert lib.fcmoe_head_norm_rope(n, None) == -1
    c = cabi.LatentAppendArgs(tokens=tokens, rot_dim=64, cache=cache, kv=4096, positions=4096, slots=4096, cos_sin=4096)
    assert lib.fcmoe_latent_cache_append(c, None) == -1
    p = cabi.HeadProjectionArgs(tokens=tokens, heads=heads, n=16, k=16, x=4096, w_packed=4096, out=4096)
    assert lib.fcmoe_head_projection(p, None) == -1
    e = cabi.ExpandedArgs(tokens=tokens, keys=1, heads=heads, batch=1, nope_dim=128, v_dim=128, scale=1.0)
    assert lib.fcmoe_expanded_attention(e, None) == -1
