"""How exact the tree operators are where their operands are cut to fewer bits.

Tolerances (u = 2^-8, half a bf16 step relative to the value): the output's rounding, u |ref|,
and what the operands' parts leave of the sum of sizes that they enter: two bf16 parts of a
probability 2^-16 at most, of the stored state 2^-17; 2^-18 more for the fp32 arithmetic
(sums of 128 to 4000 terms by fours and eights, the exponential's two units in 2^-23).
"""
import numpy as np
import pytest
import torch

import _tree_reference as R
from test_gpu_tree import DEV, U, Gdn, Paged, bf, host, i32, ops, rnd  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,HQ,HKV,nodes", [(128, 16, 4, 1), (64, 8, 2, 1), (256, 8, 2, 1), (128, 4, 1, 4),
                                           (64, 4, 2, 8)])
@pytest.mark.parametrize("ctx", [[0, 1, 40, 700], [4000]])
def test_attention_of_few_rows(ops, D, HQ, HKV, nodes, ctx):  # noqa: F811
    """Up to 16 rows of a kv-head, the decode step among them, over values whose weighted sum
    nearly cancels: what rounded probabilities would leave shows."""
    lens = [nodes] * len(ctx)
    c, trees = Paged(HKV, D, 64, ctx, lens, 5), R.make_trees(lens, 2)
    q = rnd(np.random.default_rng(1), sum(lens), HQ, D)
    out = ops.attention_tree(bf(q), c.d_k, c.d_v, c.d_table, c.d_ctx, i32(R.cu_of(lens)),
                             i32(np.concatenate(trees)), nodes, c.most)
    ref, size = R.attention(q, c.ks, c.vs, ctx, trees, D ** -0.5)
    tol = U * np.abs(ref) + (2.0 ** -16 + 2.0 ** -18) * size
    err = np.abs(host(out) - ref)
    assert (err <= tol).all(), f"{(err > tol).sum()} of {err.size}, worst {(err / tol).max():.2f}"
    assert ops.check_status() == 0


@pytest.mark.parametrize("D,nodes", [(128, 8), (64, 8), (128, 16), (64, 30), (128, 64), (64, 64)])
def test_stored_states(ops, D, nodes):  # noqa: F811
    """q over states that cancel but for their low bits: entries of 1 + 2^-8 + 2^-15 - 2^-23
    against -(1 + 2^-8).  Both parts rounded leave 2^-17 of an entry at most, both cut 2^-15."""
    c = Gdn(1, 2, D, [nodes, 1], seed=nodes, chain=True)
    c.pool[:, 1, :, 0::2] = 1 + 2.0 ** -8 + 2.0 ** -15 - 2.0 ** -23
    c.pool[:, 1, :, 1::2] = -(1 + 2.0 ** -8)
    c.y[:, :D] = 1.0                                    # q
    c.beta[:] = 0.0                                     # no node changes the state
    c.g[:] = 0.0
    c.upload()
    ref = c.delta_ref(False)
    size = D ** -0.5 * D ** 0.5 * 1.01                  # sum of |S| |q|: D entries of D^-1/2 D^-1/2
    err = np.abs(host(c.delta(ops, False)) - ref)
    tol = U * np.abs(ref) + (2.0 ** -17 + 2.0 ** -18) * size
    assert (err <= tol).all(), f"worst {(err / tol).max():.2f} of the tolerance"
