"""What is not finite in the gated delta rule along trees: value columns are independent
in the recurrence, so one element of a value, or one column of a stored state, reaches
that column of the nodes that see it and nothing else, whichever size the trees have.

Finite outputs: the tolerances of test_gpu_tree.py.
"""
import numpy as np
import pytest
import torch

import _tree_reference as R
from test_gpu_tree import Gdn, close, host, ops  # noqa: F401

pytestmark = pytest.mark.gpu


def check(got, ref, hit):
    """hit [rows, HV, D]: where the outputs cannot be finite; all others as in ref."""
    got = host(got)
    assert not np.isfinite(got[hit]).any(), "a value that is not finite went missing"
    fine = ~hit
    assert np.isfinite(got[fine]).all(), f"{(~np.isfinite(got[fine])).sum()} elements too many"
    close(np.where(hit, ref, got), ref, 2.0 ** -12)


def descendants(c, r, node):
    """Rows of the batch that see node `node` of sequence r."""
    start = sum(c.lens[:r])
    rows = np.zeros(c.N, bool)
    for i, par in enumerate(c.trees[r]):
        rows[start + i] = node in R.ancestors(c.trees[r], i)
    return rows


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("HV,D,n", [(2, 128, 7), (4, 64, 8), (2, 64, 15), (2, 128, 30), (2, 64, 64),
                                    (1, 128, 64)])
def test_one_element_of_a_value(ops, HV, D, n, bad):  # noqa: F811
    c = Gdn(1, HV, D, [3, n, 2], seed=n, wide=3)
    ref, hit = c.delta_ref(False), np.zeros((c.N, HV, D), bool)
    for node, h, col in ((1, 0, 5), (n // 2, HV - 1, D - 1), (n - 1, 0, D // 2)):
        c.d_v[3 + node, h, col] = bad
        hit[:, h, col] |= descendants(c, 1, node)
    check(c.delta(ops, False), ref, hit)
    assert ops.check_status() == 0


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("D,n", [(128, 7), (64, 16), (128, 30), (64, 40), (128, 64)])
def test_one_element_of_a_state(ops, D, n, bad):  # noqa: F811
    c = Gdn(1, 2, D, [3, n, 2], seed=n, wide=3)
    ref, hit = c.delta_ref(False), np.zeros((c.N, 2, D), bool)
    c.d_pool[c.ids[1], 1, 1, 9, 3] = bad
    hit[3:3 + n, 1, 3] = True
    check(c.delta(ops, False), ref, hit)


def test_large_finite_updates_stay(ops):  # noqa: F811
    """An update near the type's largest value is finite, and so are the outputs that a small
    decay or write strength leaves of it."""
    c = Gdn(1, 2, 64, [3], seed=1, chain=True)
    kd = 2 * 64
    c.y[:, kd:] = 0.0
    c.y[0, kd] = 3.2e38
    c.y[0] = torch.from_numpy(c.y[0]).to(torch.bfloat16).double().numpy()
    c.beta[0] = 1.0
    c.g[1:] = -40.0
    c.upload()
    got = host(c.delta(ops, False))
    ref = c.delta_ref(False)
    assert np.isfinite(ref).all() and np.isfinite(got).all()
    close(got, ref, 2.0 ** -12)


@pytest.mark.parametrize("D,n,groups", [(128, 8, 3), (128, 16, 2), (128, 30, 2), (128, 64, 1), (64, 8, 4),
                                        (64, 16, 3), (64, 32, 2), (64, 64, 1)])
def test_empty_sequences_between_nodes_that_are_not_finite(ops, D, n, groups):  # noqa: F811
    """As many heads as a CTA has groups of warps, and three units and more to each of them (148 CTAs,
    at head dim 64 two to an SM), so that a group meets a full tree, an empty one and a full one in
    turn; the last warp's columns alone hold what is not finite, so that its warps are not done at
    the same time."""
    lens = [n, 0, n - 1, 0, 0, n, 1, 0] * (60 if D == 128 else 120)
    c = Gdn(1, groups, D, lens, seed=n + D, wide=3)
    hit = np.zeros((c.N, groups), bool)
    at = 0
    for m, par in zip(lens, c.trees):
        if m > 2:
            c.d_v[at + 1, :, D - 2:] = float("inf")
            hit[at:at + m] = np.array([1 in R.ancestors(par, i) for i in range(m)])[:, None]
        at += m
    ref = c.delta_ref(False)
    for _ in range(3):
        got = host(c.delta(ops, False))
        assert not np.isfinite(got[hit][:, D - 2:]).any()
        assert np.isfinite(got[~hit]).all() and np.isfinite(got[hit][:, :D // 2]).all()
        got[hit] = ref[hit]
        close(got, ref, 2.0 ** -12)
    assert ops.check_status() == 0
