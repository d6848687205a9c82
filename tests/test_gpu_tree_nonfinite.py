"""What is not finite in the gated delta rule along trees: value columns are independent
in the recurrence, so one element of a value, or one column of a stored state, reaches
that column of the nodes that see it and nothing else, whichever size the trees have.

Finite outputs: the tolerances of test_gpu_tree.py.
"""
import numpy as np
import pytest

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
