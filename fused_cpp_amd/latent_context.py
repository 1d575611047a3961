"""Parts of a latent context on MI355X, beside ``fused_cpp_amd.latent_attention``, as HIP kernels.

* drafted tokens, a tree a sequence, appended behind its context in the nodes'
  order, at rotation positions ``context + tree.depths``:

    tree = draft_tree(parents, query_starts, max_nodes)      # once a step, for all layers
    o = absorbed_attention(..., query_starts=query_starts, tree=tree)
    latent_cache_move(cache, page_table, accepted, counts, starts=context)    # accepted: the nodes' cache positions

* a cache that keeps the tokens which the softmax weights fall on, cut down now
  and then:

    o, lse = absorbed_attention(..., return_lse=True)
    attention_weights(q_latent, q_rope, cache, page_table, kv_lens, lse, scale=..., previous=weights, out=weights)
    positions, kept, kept_weights = heaviest_positions(weights, kv_lens, keep, sinks=4, recent=128)
    latent_cache_move(cache, page_table, positions, kept)    # kept: the new kv_lens
    n = min(keep, weights.shape[1])
    weights.zero_()[:, :n] = kept_weights[:, :n]             # the rows' sums move with them

Scores, weights and their sums are fp32. Streams, capture into HIP graphs, errors,
and what written tensors may share are ``latent_attention``'s; inputs that require a
gradient are refused while gradients are recorded, and inputs with a forward-mode tangent.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from fused_cpp_amd import _native
from fused_cpp_amd.latent_attention import DraftTree, LatentCache


def draft_tree(parents: torch.Tensor, query_starts: torch.Tensor, max_nodes: int) -> DraftTree:
    """The masks and depths of drafted trees, for :func:`~fused_cpp_amd.latent_attention.absorbed_attention`.

    ``parents [T]`` int32: of each sequence's nodes (``query_starts [B + 1]`` int32, as there) the parent's number
    among them, which lies below the node's own; any other value (-1) makes it a root, a child of the sequence's last
    token. A node sees itself and its ancestors. ``max_nodes`` (1 to 1024) bounds the nodes of a sequence: ones past
    it, rounded up to 64, get no bits and depth 0, as tokens of no sequence do.
    """
    masks, depths = _native.require_native().latent_draft_tree(parents, query_starts, max_nodes)
    return DraftTree(masks, depths)


def attention_weights(q_latent: torch.Tensor, q_rope: Optional[torch.Tensor], cache: LatentCache,
                      page_table: torch.Tensor, kv_lens: torch.Tensor, lse: torch.Tensor, *, scale: float,
                      query_starts: Optional[torch.Tensor] = None, previous: Optional[torch.Tensor] = None,
                      out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """What each cached token received of a call's softmax weights, summed over its query tokens and heads, added to
    ``previous``: ``[B, positions]`` fp32 by position in the sequence.

    The queries, cache and lengths of a causal :func:`~fused_cpp_amd.latent_attention.absorbed_attention` and the
    ``lse`` that it returned. Positions are ``previous``'s (or ``out``'s) columns, else the page table's reach; tokens
    past them are left out, and places past a length keep what they had (0 without ``previous``). ``out`` may be
    ``previous`` itself. A query whose lse is -inf adds nothing, whatever its row holds; a page id outside the cache makes
    the weights of its tokens that other queries see NaN. Sums are taken in fp32, in an order that only the shapes and
    lengths decide.
    """
    return _native.require_native().latent_attention_weights(
        q_latent, q_rope, cache.latent, cache.rope, cache.scale, page_table, kv_lens, lse, scale, query_starts,
        previous, out)


def heaviest_positions(weights: torch.Tensor, kv_lens: torch.Tensor, keep: int, *, sinks: int = 0, recent: int = 0
                       ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The positions that stay when every sequence keeps ``keep`` of its tokens: ``(positions, counts, weights)``.

    Of a sequence with more of them its first ``sinks``, its last ``recent``, and of the others those with the
    largest ``weights [B, positions]`` fp32 (ties go to the lower position, NaN counts as the largest); of a shorter
    one all. ``positions [B, keep]`` int32 ascends, with -1 behind ``counts [B]`` int32; the weights there come
    back beside them, 0 behind. Lengths ``kv_lens [B]`` int32 are cut to the columns there are.
    """
    return _native.require_native().latent_heaviest_positions(weights, kv_lens, keep, sinks, recent)


def latent_cache_move(cache: LatentCache, page_table: torch.Tensor, positions: torch.Tensor, counts: torch.Tensor, *,
                      starts: Optional[torch.Tensor] = None, to_table: Optional[torch.Tensor] = None) -> None:
    """Moves cached rows (with their key parts and scales): row ``positions[b, k]`` of sequence b becomes its row
    ``starts[b] + k`` (``k`` without ``starts``), for ``k < counts[b]``. All are int32.

    Without ``to_table`` the rows stay in the sequence's own pages: ``positions[b]`` then has to ascend with
    ``positions[b, k] >= starts[b] + k``, as those of :func:`heaviest_positions` and of accepted drafts do, and no
    other sequence may share the pages that are written. With ``to_table [B, pages]`` they go to that table's pages, in
    any order, which must hold no row that the call reads. A row whose position at either end names no cached row (-1,
    past the table, a page id outside the cache) is left out.
    """
    _native.require_native().latent_cache_move(cache.latent, cache.rope, cache.scale, page_table, positions, counts,
                                               starts, to_table)


__all__ = [
    "DraftTree",
    "attention_weights",
    "draft_tree",
    "heaviest_positions",
    "latent_cache_move",
]
