"""Bounded waits of the tree operators that run out: with the poll limit lowered (the test
hook gdn_set_wait_limit) a call gives up, says so in the status word, and leaves the outputs
that it could not compute as they were; the next call is right again.

Limit 0: no wait succeeds, nothing is written.  Small limits: some do, and what is written is
right.  Tolerances of test_gpu_tree.py.
"""
import numpy as np
import pytest
import torch

import _tree_reference as R
from test_gpu_tree import DEV, U, Gdn, Paged, attn_close, bf, close, host, i32, ops, rnd  # noqa: F401

pytestmark = pytest.mark.gpu
LEFT = 7.0


def run_short_of(ops, polls, call):  # noqa: F811
    """call() under a limit; whether it gave up."""
    ops.check_status()
    ops.set_wait_limit(polls)
    try:
        call()
        torch.cuda.synchronize()
    finally:
        ops.set_wait_limit(None)
    try:
        ops.check_status()
    except ops._lib.GdnError as e:
        assert "wait" in str(e)
        return True
    return False


def check_units(got, ref, slack):
    """got / ref [rows, heads, D]: every head of a row either as it was or right."""
    left = (got == LEFT).all(-1)
    tol = U * np.abs(ref) + slack + 1e-30
    assert (left | (np.abs(got - ref) <= tol).all(-1)).all()
    return left


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("D,n", [(128, 8), (128, 16), (128, 30), (128, 64), (64, 8), (64, 16), (64, 32), (64, 64)])
def test_delta_rule_that_gives_up(ops, D, n, norm):  # noqa: F811
    r = np.random.default_rng(n + D)
    lens = [int(x) for x in r.integers(0, n + 1, 200)]
    lens[0], lens[3] = n, 0
    c = Gdn(1, 4, D, lens, seed=n)
    ref = c.delta_ref(norm)
    slack = 2.0 ** -12 * np.abs(ref).max(-1, keepdims=True)
    pool = c.d_pool.clone()
    for polls in (0, 1, 2, 3, 5, 8, 20):
        out = torch.full((c.N, 4, D), LEFT, dtype=torch.bfloat16, device=DEV)
        gave_up = run_short_of(ops, polls, lambda: c.delta(ops, norm, out=out))
        left = check_units(host(out), ref, slack)
        assert gave_up or not left.any()
        if polls == 0:
            assert gave_up and left.all()
        assert torch.equal(c.d_pool, pool)
        close(c.delta(ops, norm), ref, 2.0 ** -12, "the next call")
        assert ops.check_status() == 0


@pytest.mark.parametrize("D,nodes,HQ,HKV", [
    (128, 1, 8, 2), (64, 1, 8, 2), (256, 1, 4, 1),      # 16 rows of a unit
    (128, 8, 4, 1), (64, 8, 4, 1), (256, 8, 4, 1),      # 32
    (128, 40, 4, 1), (64, 40, 4, 2), (256, 40, 4, 1),   # 128; 64 at head dim 256
    (128, 64, 8, 1)])                                   # several row tiles
@pytest.mark.parametrize("many", [False, True])
def test_attention_that_gives_up(ops, D, nodes, HQ, HKV, many):  # noqa: F811
    """Few long sequences, whose units are all cut and joined, and many short ones."""
    r = np.random.default_rng(nodes + D)
    ctx = [int(x) for x in r.integers(0, 400, 90)] if many else [6000, 37, 2500]
    lens = [int(x) for x in r.integers(0, nodes + 1, len(ctx))]
    lens[0] = nodes
    if many:
        lens = [n if i % 6 == 0 else min(n, 3) for i, n in enumerate(lens)]
    c, trees = Paged(HKV, D, 32, ctx, lens, 3), R.make_trees(lens, 1)
    n = sum(lens)
    q = rnd(r, n, HQ, D)
    ref, size = R.attention(q, c.ks, c.vs, ctx, trees, D ** -0.5)
    args = (bf(q), c.d_k, c.d_v, c.d_table, c.d_ctx, i32(R.cu_of(lens)), i32(np.concatenate(trees)),
            nodes, c.most)
    for polls in (0, 1, 2, 3, 5, 8, 20, 100):
        out = torch.full((n, HQ, D), LEFT, dtype=torch.bfloat16, device=DEV)
        gave_up = run_short_of(ops, polls, lambda: ops.attention_tree(*args, out=out))
        left = check_units(host(out), ref, U * size)
        assert gave_up or not left.any()
        if polls == 0:
            assert gave_up and left.all()
        attn_close(ops.attention_tree(*args), ref, size)
        assert ops.check_status() == 0
