"""Latent attention on MI355X: the steps between the W8A8 attention projections
(``fused_cpp_amd.deepseek_v4_w8a8``) of a DeepSeek layer, as HIP kernels.

One latent row a token (``latent_dim`` values that all heads share as keys and
values, ``rope_dim`` rotated key values beside them) lies in a paged cache:

    q = deepseek_v4_w8a8_linear(...)                         # [T, H, nope + rope]
    head_norm_rope(q, positions, cos_sin, normalize=False, out=q)
    latent_cache_append(kv, positions, slots, cos_sin, cache, weight=kv_norm)

* decode, absorbed form: queries go into the latent space, attention reads the
  cache itself, outputs come back per head:

    q_latent = head_projection(q[..., :nope], w_uk)
    o = absorbed_attention(q_latent, q[..., nope:], cache, page_table, kv_lens, scale=...)
    values = head_projection(o, w_uv)                        # into wo_b

* prompts, expanded form, over the up-projected keys and values:

    rows = latent_cache_append(..., return_rows=True)
    values = expanded_attention(q, kv_up, rows[:, latent_dim:], query_starts, scale=...)

Everything is bf16 in and out. Norms, rotations, scores, softmax sums and all
accumulators are fp32; the attentions round each softmax weight once to bf16 for
its product with the values (times its token's scale in an e4m3 cache). The cache
is bf16, or e4m3 with one fp32 scale a token. Inference only: inputs that require
a gradient are refused while gradients are recorded, and inputs with a forward-mode
tangent; an ``out`` or a cache that is written counts as changed in place. Calls
run on the current stream of their tensors' device, allocate through torch, read
lengths, positions, slots and page ids on the device only, and can be captured into
a HIP graph. What a call writes may lie between the rows of what it reads, as views
of one tensor do, but share no memory with it.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from fused_cpp_amd import _native


@dataclass(frozen=True)
class LatentCache:
    """A paged cache of latent rows; token slot ``s`` is row ``s % page_size`` of page ``s // page_size``.

    ``latent [pages, page_size, latent_dim]`` and ``rope [pages, page_size, rope_dim]`` (``None`` without a separate
    key part) are bf16, or ``float8_e4m3fn`` with ``scale [pages, page_size]`` fp32: a value is its byte times its
    token's scale. ``latent_dim`` is 256 or 512, ``rope_dim`` 64 or none. Rows have to start at multiples of 16
    bytes, so both may be views of one ``[pages, page_size, latent_dim + rope_dim]`` tensor.
    """

    latent: torch.Tensor
    rope: Optional[torch.Tensor] = None
    scale: Optional[torch.Tensor] = None


def allocate_latent_cache(pages: int, page_size: int, *, latent_dim: int = 512, rope_dim: int = 64,
                          dtype: torch.dtype = torch.bfloat16, device=None) -> LatentCache:
    """A zeroed :class:`LatentCache`; ``dtype`` bfloat16, or float8_e4m3fn (which adds the scales)."""
    if dtype not in (torch.bfloat16, torch.float8_e4m3fn):
        raise TypeError(f"cache dtype must be bfloat16 or float8_e4m3fn, got {dtype}")
    if latent_dim not in (256, 512) or rope_dim not in (0, 64):
        raise ValueError(f"latent_dim must be 256 or 512 and rope_dim 0 or 64, got {latent_dim} and {rope_dim}")
    if pages < 0 or page_size <= 0:
        raise ValueError(f"need pages >= 0 and page_size > 0, got {pages} and {page_size}")
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)

    def zeros(dim):
        return torch.zeros((pages, page_size, dim), dtype=torch.uint8 if dtype != torch.bfloat16 else dtype,
                           device=device).view(dtype)

    return LatentCache(zeros(latent_dim), zeros(rope_dim) if rope_dim else None,
                       torch.zeros((pages, page_size), device=device) if dtype != torch.bfloat16 else None)


@dataclass(frozen=True)
class PreparedHeadProjection:
    """Per-head weights ``[heads, n, k]`` in the kernels' operand order."""

    packed: torch.Tensor
    heads: int
    n: int
    k: int


def head_norm_rope(x: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor, *,
                   weight: Optional[torch.Tensor] = None, eps: float = 1e-6, normalize: bool = True,
                   inverse: bool = False, interleaved: bool = True, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """RMS norm of each head of ``x [T, H, D]`` and rotation of its last values, in one pass.

    ``x * rsqrt(mean(x^2) + eps) * weight`` (``normalize``; ``weight [D]`` optional), then the last
    ``cos_sin.shape[1]`` values of a head turn by the angles of table row ``positions[t]``: ``cos_sin
    [positions, rope_dim]`` fp32 holds the cosines of the pairs, then their sines. Pairs are neighbours
    (``interleaved``) or half the rotated part apart; ``inverse`` turns back. A position outside the table makes the
    rotated values NaN. ``out`` may be ``x`` itself.
    """
    return _native.require_native().latent_head_norm_rope(x, positions, cos_sin, weight, eps, normalize, inverse,
                                                          interleaved, out)


def latent_cache_append(kv: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor, cos_sin: torch.Tensor,
                        cache: LatentCache, *, weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                        interleaved: bool = True, return_rows: bool = False) -> Optional[torch.Tensor]:
    """Writes latent rows into the cache, normalised and rotated on the way.

    ``kv [T, latent_dim + rope_dim]``: the first ``latent_dim`` values are RMS-normalised (times ``weight``), the last
    ``cos_sin.shape[1]`` values rotated as in :func:`head_norm_rope` (``rope_dim`` of them; with no separate key part
    any multiple of 16 of the latent's). An e4m3 cache takes ``max|row| / 448`` as the row's scale. A token whose slot
    lies outside the cache (-1 for padding) is not written. The slots of a call have to differ: one given twice ends
    up with either row or a mixture of them. ``return_rows`` returns the rows ``[T, latent_dim + rope_dim]`` in bf16
    as well, every token's: the expanded form's inputs.
    """
    return _native.require_native().latent_cache_append(kv, positions, slots, cos_sin, cache.latent, cache.rope,
                                                        cache.scale, weight, eps, interleaved, return_rows)


def prepare_head_projection(weight: torch.Tensor) -> PreparedHeadProjection:
    """Packs per-head weights ``[H, N, K]`` bf16 (any strides) for :func:`head_projection`; N and K multiples of 8."""
    packed, heads, n, k = _native.require_native().latent_prepare_head_projection(weight)
    return PreparedHeadProjection(packed=packed, heads=int(heads), n=int(n), k=int(k))


def head_projection(x: torch.Tensor, weight: PreparedHeadProjection, *, out: Optional[torch.Tensor] = None
                    ) -> torch.Tensor:
    """``out[t, h] = weight[h] @ x[t, h]``: ``x [T, H, K]`` (rows at multiples of 16 bytes are read in place) to
    ``[T, H, N]``."""
    if not isinstance(weight, PreparedHeadProjection):
        raise TypeError("weight must come from prepare_head_projection")
    return _native.require_native().latent_head_projection(x, weight.packed, weight.heads, weight.n, weight.k, out)


def absorbed_attention(q_latent: torch.Tensor, q_rope: Optional[torch.Tensor], cache: LatentCache,
                       page_table: torch.Tensor, kv_lens: torch.Tensor, *, scale: float,
                       query_starts: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                       return_lse: bool = False):
    """Attention of queries in the latent space over the paged cache: ``[T, H, latent_dim]``.

    ``q_latent [T, H, latent_dim]`` and ``q_rope [T, H, rope_dim]`` (``None`` without a separate key part).
    ``page_table [B, width]`` int32, ``kv_lens [B]`` int32: cached tokens of each sequence, this call's included.
    ``query_starts [B + 1]`` int32: sequence b's query tokens; without it each sequence has one. Starts are cut to the
    tokens there are, and one below an earlier one counts as that one: a batch may be padded with any of either. Query
    i of n sees the first ``kv_lens[b] - n + i + 1`` tokens; one that sees none is 0. Lengths past the table's reach are
    cut to it, a page id outside the cache makes its sequence NaN. Cached tokens that a sequence's queries do not all
    see have to be finite; rows past a length may hold anything.

    ``return_lse`` adds ``[T, H]`` fp32: the log of the softmax's sum (-inf where there is none), which joins results
    over parts of a context. Tokens that no sequence holds are 0, or left as they were in a given ``out``.
    """
    o, lse = _native.require_native().latent_absorbed_attention(
        q_latent, q_rope, cache.latent, cache.rope, cache.scale, page_table, kv_lens, query_starts, scale, out,
        return_lse)
    return (o, lse) if return_lse else o


def expanded_attention(q: torch.Tensor, kv: torch.Tensor, k_rope: Optional[torch.Tensor], query_starts: torch.Tensor,
                       *, scale: float, kv_starts: Optional[torch.Tensor] = None, causal: bool = True,
                       out: Optional[torch.Tensor] = None, return_lse: bool = False):
    """Attention over per-head keys and values ``kv [S, H, nope + v]`` and a key part ``k_rope [S, rope_dim]`` that
    the heads share (``None`` without one): ``[T, H, v]`` from ``q [T, H, nope + rope_dim]``.

    Sequences are packed: ``query_starts [B + 1]`` and ``kv_starts [B + 1]`` int32 (default: the same) bound their
    query tokens and keys, query starts as in :func:`absorbed_attention`. With ``causal`` query i of n sees the
    first ``keys - n + i + 1`` keys. ``nope`` and ``v`` are both 128 or both 64, ``rope_dim`` 64 or none. Keys and values
    that a sequence's queries do not all see have to be finite; what no sequence holds may be anything. Empty rows,
    ``return_lse`` and ``out`` as in :func:`absorbed_attention`.
    """
    o, lse = _native.require_native().latent_expanded_attention(q, kv, k_rope, query_starts, kv_starts, scale, causal,
                                                                out, return_lse)
    return (o, lse) if return_lse else o


__all__ = [
    "LatentCache",
    "PreparedHeadProjection",
    "absorbed_attention",
    "allocate_latent_cache",
    "expanded_attention",
    "head_norm_rope",
    "head_projection",
    "latent_cache_append",
    "prepare_head_projection",
]
