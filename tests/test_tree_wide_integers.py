"""Metadata given as 64-bit integers: what 32 bits cannot hold is as wrong as before and never
wraps around to a value that looks right."""
import numpy as np
import pytest
import torch

WIDE = [2 ** 32 + 3, -2 ** 32, 2 ** 31, -2 ** 31 - 1, 2 ** 62]


def test_narrowing_saturates(pkg):
    t = torch.tensor(WIDE + [5, -1])
    got = pkg.ops._int32(t, 7, "t").tolist()
    assert got == [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, 5, -1]
    with pytest.raises(AssertionError, match="integers"):
        pkg.ops._int32(t.double(), 7, "t")


@pytest.fixture(scope="module")
def ops(pkg):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.set_device(0)
    return pkg.ops


def flagged(ops, error):
    with pytest.raises(error):
        ops.check_status()
    assert ops.check_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("wide", WIDE)
def test_wide_metadata_is_flagged(ops, wide):
    from test_gpu_tree import DEV, Gdn, bf, f32, i32, i64, rnd
    r = np.random.default_rng(0)
    d, w = bf(rnd(r, 2, 4, 64)), bf(np.ones(64))
    kc, vc = (torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    cs = f32(np.concatenate([np.ones((8, 16)), np.zeros((8, 16))], 1))
    ops.qk_norm_rope_cache(d[:, :2], d[:, 2:3], d[:, 3:], w, w, cs, i64([0, 1]), kc, vc, i64([wide, 7]))
    flagged(ops, IndexError)
    assert (kc.view(8, 64)[:7] == 0).all() and (vc.view(8, 64)[:7] == 0).all()
    c = Gdn(1, 2, 64, [4, 2], seed=1)
    pool, conv = c.d_pool.clone(), c.d_conv.clone()
    args = (c.d_x, c.d_k, c.d_v, c.d_g, c.d_beta, c.d_conv[:, 1], c.d_pool[:, 1], c.d_ids)
    ops.commit_tree(*args, *c.tree, i64([wide, -1]))
    flagged(ops, ValueError)
    ops.commit_tree(*args, c.d_cu, i64([-1, wide, 0, 0, -1, 0]), 4, i32([3, -1]))
    flagged(ops, ValueError)
    ops.commit_tree(*args, i64([0, 4, wide]), c.d_par, 4, i32([-1, 1]))
    flagged(ops, ValueError)
    assert torch.equal(c.d_pool, pool) and torch.equal(c.d_conv, conv)
    table, q = i32([[0, 1], [1, 0]]), c.d_v[:, :2].contiguous()
    out = torch.full((6, 2, 64), 7.0, dtype=torch.bfloat16, device=DEV)
    ops.attention_tree(q, kc, vc, table, i64([wide, 1]), *c.tree, 8, out=out)
    flagged(ops, ValueError)
    assert (out[:4] == 7).all() and not (out[4:] == 7).all()
