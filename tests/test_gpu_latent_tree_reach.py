"""GPU trees of drafts at the ends of what their masks and depths say: nodes that no mask has a bit for, and depths that no
tree of the call's nodes has."""

from __future__ import annotations

import pytest
import torch

from tests import context_reference as cref
from tests import latent_reference as ref
from tests.test_gpu_latent_attention import BF16, E4M3, _i32, _la, _Paged, _queries
from tests.test_gpu_latent_context import _forget, _lc, _starts, _tree_parents

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("H,singles", [(1, 50), (2, 50), (4, 50), (1, 0), (16, 0), (128, 0)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (50, 3)])
def test_nodes_past_the_masks_may_be_gone(gpu, H, singles, dtype, window, sinks):
    """Neither the rows nor the pages of nodes that the masks have no words for are read: whole tiles of such nodes and ends of
    tiles, more nodes than cached tokens. The nodes themselves see the context. Row groups go by the mean of a sequence's
    rows: 16, 32 and 64 with sequences of one node around, 128 without."""
    la, lc = _la(), _lc()
    trees = [_tree_parents("random", 90, 2), _tree_parents("chain", 300, 1), _tree_parents("star", 64, 3), _tree_parents("binary", 65, 4),
             _tree_parents("random", 200, 5), _tree_parents("chain", 100, 6)] + [[-1]] * singles
    lens = [90 + 33, 300 + 64, 64 + 7, 65 + 63, 200, 80] + [1 + 5 * k for k in range(singles)]
    pg = _Paged(H, lens, 512, 64, dtype, page=16)
    new = [len(p) for p in trees]
    assert (singles == 0) == (-(-sum(new) // len(new)) * H > 64)
    st = _i32(_starts(new))
    ql, qr = _queries(3, sum(new), H, 512, 64)
    tree = lc.draft_tree(_i32([v for p in trees for v in p]), st, 60)
    assert tree.masks.shape[1] == 1
    keeps = [cref.seen_by_tree(p, L, window, sinks, 1) for p, L in zip(trees, lens)]
    want, wl, tol, ltol = cref.absorbed(ql, qr, pg.rows, _starts(new), 0.07, keeps)
    _forget(pg, lens, keeps)
    out, lse = la.absorbed_attention(ql, qr, pg.cache, pg.table, pg.lens, scale=0.07, query_starts=st, tree=tree, window=window,
                                     sinks=sinks, return_lse=True)
    ref.assert_within(out, want, tol, "out")
    ref.assert_within(lse, wl, ltol, "lse")


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("H", [1, 4, 6, 12, 16, 128])
def test_depths_count_as_ones_of_the_nodes(gpu, H, dtype):
    """Depths of a user's own below 0 count as 0, ones past the last node's number as that. (Row groups of 16, 32, 64, 128.)"""
    la, lc = _la(), _lc()
    given = [[0, -1, 3, 2 ** 31 - 1], [-2 ** 31, 200, 1], [70], [-7, 9, 5, 4, 3, 2, 1, 0, 100]]
    context, (window, sinks) = [400, 130, 65, 200], (70, 3)
    new = [len(d) for d in given]
    lens = [c + n for c, n in zip(context, new)]
    pg = _Paged(H, lens, 512, 64, dtype, page=16)
    st = _i32(_starts(new))
    ql, qr = _queries(4, sum(new), H, 512, 64)
    masks = torch.tensor([[1 << i] for n in new for i in range(n)], dtype=torch.int64, device="cuda")
    keeps = []
    for c, d in zip(context, given):
        n, j = len(d), torch.arange(c + len(d), device="cuda")
        at = torch.tensor([c + min(max(v, 0), n - 1) for v in d], device="cuda")[:, None]
        keeps.append(((j < c) & ((j > at - window) | (j < sinks))) | (j == c + torch.arange(n, device="cuda")[:, None]))
    want, wl, tol, ltol = cref.absorbed(ql, qr, pg.rows, _starts(new), 0.07, keeps)
    out, lse = la.absorbed_attention(ql, qr, pg.cache, pg.table, pg.lens, scale=0.07, query_starts=st, window=window, sinks=sinks,
                                     tree=lc.DraftTree(masks, _i32([v for d in given for v in d])), return_lse=True)
    ref.assert_within(out, want, tol, "out")
    ref.assert_within(lse, wl, ltol, "lse")
