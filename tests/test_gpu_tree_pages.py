"""A sequence with a page that is not there: flagged, never read, and every output of the
sequence is NaN, so that nothing which another sequence left in the chip's memory shows
through; the other sequences as always."""
import numpy as np
import pytest
import torch

import _tree_reference as R
from test_gpu_tree import DEV, Paged, attn_close, bf, i32, ops, rnd  # noqa: F401
from test_gpu_tree_faults import flagged, rows_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nodes,D,HQ,HKV", [(1, 128, 2, 1), (2, 128, 4, 2), (9, 128, 2, 1), (40, 128, 2, 1),
                                            (40, 64, 4, 2), (9, 64, 2, 1), (1, 256, 2, 1), (33, 256, 2, 1)])
@pytest.mark.parametrize("ctx1,where,page", [(300, 5, -1), (300, 0, 10 ** 6), (40, 2, -7), (4000, 240, -1),
                                             (0, 0, -1)])
def test_missing_pages_give_nan(ops, nodes, D, HQ, HKV, ctx1, where, page):  # noqa: F811
    ctx, lens = [40, ctx1, 20, 64], [nodes, nodes, 1, nodes]
    c, trees = Paged(HKV, D, 16, ctx, lens, 3), R.make_trees(lens, 1)
    q = rnd(np.random.default_rng(0), sum(lens), HQ, D)
    ref, size = R.attention(q, c.ks, c.vs, ctx, trees, D ** -0.5)
    c.d_table[1, where] = page
    args = (bf(q), c.d_k, c.d_v, c.d_table, c.d_ctx, i32(R.cu_of(lens)), i32(np.concatenate(trees)),
            nodes, c.most)
    for _ in range(2):
        out = torch.zeros(sum(lens), HQ, D, dtype=torch.bfloat16, device=DEV)
        ops.attention_tree(*args, out=out)
        flagged(ops, IndexError)
        assert out[rows_of(lens, 1)].isnan().all()
        for r in (0, 2, 3):
            attn_close(out[rows_of(lens, r)], ref[rows_of(lens, r)], size[rows_of(lens, r)])


@pytest.mark.parametrize("nodes", [2, 40])
def test_short_tables_give_nan(ops, nodes):  # noqa: F811
    ctx, lens = [40, 300, 20], [nodes, nodes, 1]
    c, trees = Paged(1, 128, 16, ctx, lens, 3), R.make_trees(lens, 1)
    q = rnd(np.random.default_rng(0), sum(lens), 2, 128)
    ref, size = R.attention(q, c.ks, c.vs, ctx, trees, 128 ** -0.5)
    out = ops.attention_tree(bf(q), c.d_k, c.d_v, c.d_table[:, :10].contiguous(), c.d_ctx,
                             i32(R.cu_of(lens)), i32(np.concatenate(trees)), nodes, c.most)
    flagged(ops, IndexError)
    assert out[rows_of(lens, 1)].isnan().all()
    for r in (0, 2):
        attn_close(out[rows_of(lens, r)], ref[rows_of(lens, r)], size[rows_of(lens, r)])
