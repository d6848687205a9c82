"""A row whose position lies outside the rotation table stores nothing: its key cannot be
rotated, and a slot with a new value beside an old key would belong to no token."""
import numpy as np
import pytest
import torch

import _tree_reference as R
from test_gpu_tree import DEV, bf, close, f32, host, i32, i64, ops, rnd  # noqa: F401
from test_gpu_tree_faults import flagged

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,D,HKV", [(7, 64, 1), (40, 128, 3), (900, 128, 2)])
def test_a_bad_position_leaves_its_slot_alone(ops, n, D, HKV):  # noqa: F811
    r = np.random.default_rng(n)
    d = bf(rnd(r, n, 4 + 2 * HKV, D))
    blocks = n // 16 + 2
    kv = bf(rnd(r, 2, blocks, 16, HKV, D))
    before, w = kv.clone(), bf(np.ones(D))
    cs = f32(np.concatenate([np.ones((50, 16)), np.zeros((50, 16))], 1))
    pos, slot = r.integers(0, 50, n), r.permutation(blocks * 16)[:n]
    bad = np.zeros(n, bool)
    bad[[1, 4, n - 1]] = True
    pos[1], pos[4], pos[n - 1] = 50, -1, 1 << 40
    ops.qk_norm_rope_cache(d[:, :4], d[:, 4:4 + HKV], d[:, 4 + HKV:], w, w, cs, i64(pos), kv[0], kv[1],
                           i32(slot))
    flagged(ops, IndexError)
    k, v = (t.view(-1, HKV, D) for t in kv)
    for t, old in zip((k, v), before):
        assert torch.equal(t[slot[bad]], old.view(-1, HKV, D)[slot[bad]])
    assert torch.equal(v[slot[~bad]], d[:, 4 + HKV:][torch.from_numpy(~bad)])
    ref = R.norm_rope(host(d[:, 4:4 + HKV]), np.ones(D), np.ones((n, 16)), np.zeros((n, 16)), 1e-6, 0)
    close(k[slot[~bad]], ref[~bad], 2.0 ** -18)
