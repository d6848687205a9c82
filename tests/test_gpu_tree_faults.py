"""What the tree operators do with bad metadata on the device (flagged, never read out
of bounds, the other sequences as always), with empty calls, and with pools and
caches whose offsets pass 2^31 elements."""
import numpy as np
import pytest
import torch

import _tree_reference as R
from test_gpu_tree import DEV, U, Gdn, Paged, attn_close, bf, close, f32, host, i32, i64, ops, rnd  # noqa: F401

pytestmark = pytest.mark.gpu


def rows_of(lens, r):
    return slice(sum(lens[:r]), sum(lens[:r + 1]))


def flagged(ops, error):  # noqa: F811
    with pytest.raises(error):
        ops.check_status()
    assert ops.check_status() == 0


BAD_CU = [
    ([0, 4, 2, 9, 12], [1]),            # a negative length: the next one reads what it says
    ([0, 4, 9, 20, 12], [2, 3]),        # past the rows, then negative
    ([0, 4, 12, 12, 12], [1]),          # eight rows where five are allowed
    ([-3, 4, 9, 12, 12], [0]),          # a negative start
]


@pytest.mark.parametrize("cu,bad", BAD_CU)
def test_malformed_cu_seqlens(ops, cu, bad):  # noqa: F811
    lens = [4, 5, 3, 0]
    c = Gdn(1, 2, 64, lens, seed=3)
    ref = c.delta_ref(False)
    c.d_cu = i32(cu)
    c.tree = (c.d_cu, c.d_par, 5)
    pool, conv = c.d_pool.clone(), c.d_conv.clone()
    out = torch.full((c.N, 2, 64), 9.0, dtype=torch.bfloat16, device=DEV)
    c.delta(ops, False, out=out)
    flagged(ops, ValueError)
    for r in range(3):
        if r not in bad and cu[r:r + 2] == R.cu_of(lens)[r:r + 2].tolist():
            close(out[rows_of(lens, r)], ref[rows_of(lens, r)], 2.0 ** -12)
    c.commit(ops, [3, 4, 2, -1])
    flagged(ops, ValueError)
    for r in bad:
        s = c.ids[r]
        assert torch.equal(c.d_pool[s], pool[s]) and torch.equal(c.d_conv[s], conv[s])
    ops.conv_gate_tree(c.d_x, c.d_conv[:, 1], c.d_ids, bf(c.w), *c.tree, c.d_b, c.d_a, f32(c.a_log),
                       f32(c.dt))
    ops.tree_slot_map(i32(np.arange(8).reshape(4, 2)), i32([0, 0, 0, 0]), *c.tree, 16, c.N)
    kc, vc = (torch.zeros(8, 16, 1, 64, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    q = torch.zeros(c.N, 2, 64, dtype=torch.bfloat16, device=DEV)
    ops.attention_tree(q, kc, vc, i32(np.arange(8).reshape(4, 2)), i32([0, 0, 0, 0]), *c.tree, 32)
    flagged(ops, ValueError)


@pytest.mark.parametrize("cu", [c for c, _ in BAD_CU])
def test_every_operator_flags_malformed_cu_seqlens(ops, cu):  # noqa: F811
    c = Gdn(1, 2, 64, [4, 5, 3, 0], seed=3)
    tree = (i32(cu), c.d_par, 5)
    kc, vc = (torch.zeros(8, 16, 1, 64, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    q, table, ctx = c.d_v[:, :2].contiguous(), i32(np.arange(8).reshape(4, 2)), i32([0] * 4)
    calls = [
        lambda: ops.conv_gate_tree(c.d_x, c.d_conv[:, 1], c.d_ids, bf(c.w), *tree, c.d_b, c.d_a,
                                   f32(c.a_log), f32(c.dt)),
        lambda: ops.gated_delta_rule_tree(c.d_q, c.d_k, c.d_v, c.d_g, c.d_beta, c.d_pool[:, 1],
                                          c.d_ids, *tree),
        lambda: ops.commit_tree(c.d_x, c.d_k, c.d_v, c.d_g, c.d_beta, c.d_conv[:, 1], c.d_pool[:, 1],
                                c.d_ids, *tree, i32([0, 0, 0, -1])),
        lambda: ops.tree_slot_map(table, ctx, *tree, 16, c.N),
        lambda: ops.attention_tree(q, kc, vc, table, ctx, *tree, 32),
        lambda: ops.attention_tree(q.repeat(1, 8, 1), kc, vc, table, ctx, *tree, 32),
    ]
    for call in calls:
        call()
        flagged(ops, ValueError)


@pytest.mark.parametrize("row,parent", [(2, 2), (1, 7), (3, -5), (0, 0), (4, 1 << 30), (3, -(1 << 31))])
def test_malformed_parents(ops, row, parent):  # noqa: F811
    lens = [5, 20, 6]
    c = Gdn(1, 2, 128, lens, seed=3)
    ref = c.delta_ref(True)
    c.d_par[5 + row] = parent
    pool, conv = c.d_pool.clone(), c.d_conv.clone()
    out = c.delta(ops, True)
    flagged(ops, ValueError)
    for r in (0, 2):
        close(out[rows_of(lens, r)], ref[rows_of(lens, r)], 2.0 ** -12)
    c.commit(ops, [4, 19, 5])
    flagged(ops, ValueError)
    s = c.ids[1]
    assert torch.equal(c.d_pool[s], pool[s]) and torch.equal(c.d_conv[s], conv[s]), "left alone"
    c.d_pool[s], c.d_conv[s] = pool[s], conv[s]
    acc = [4, -1, 5]
    win, st = c.commit_ref(acc)
    for r in (0, 2):
        assert np.array_equal(host(c.d_conv)[c.ids[r], 1], win[r])
        assert np.linalg.norm(host(c.d_pool)[c.ids[r], 1] - st[r]) <= 1e-5 * np.linalg.norm(st[r])
    pos, slot = ops.tree_slot_map(i32(np.arange(30).reshape(3, 10)), i32([3, 4, 5]), *c.tree, 16, c.N,
                                  accepted=i32(acc))
    flagged(ops, ValueError)
    rp, rs = R.slots(np.arange(30).reshape(3, 10), [3, 4, 5], c.trees, 16, acc)
    for r in (0, 2):
        assert np.array_equal(pos[rows_of(lens, r)].cpu().numpy(), rp[rows_of(lens, r)])
        assert np.array_equal(slot[rows_of(lens, r)].cpu().numpy(), rs[rows_of(lens, r)])
    ops.conv_gate_tree(c.d_x, c.d_conv[:, 1], c.d_ids, bf(c.w), *c.tree, c.d_b, c.d_a, f32(c.a_log),
                       f32(c.dt))
    flagged(ops, ValueError)


@pytest.mark.parametrize("accepted", [[5, 0], [-2, 0], [1 << 30, 0]])
def test_accepted_nodes_that_are_not_there(ops, accepted):  # noqa: F811
    c = Gdn(1, 2, 64, [5, 2], seed=1)
    pool, conv = c.d_pool.clone(), c.d_conv.clone()
    c.commit(ops, accepted)
    flagged(ops, ValueError)
    s = c.ids[0]
    assert torch.equal(c.d_pool[s], pool[s]) and torch.equal(c.d_conv[s], conv[s])
    pos, slot = ops.tree_slot_map(i32([[0], [1]]), i32([0, 0]), *c.tree, 16, c.N,
                                  accepted=i32(accepted))
    flagged(ops, ValueError)
    assert (slot[:5] == -1).all() and slot[5:].tolist() == [16, -1]


def test_slots_outside_the_pool(ops):  # noqa: F811
    c = Gdn(1, 2, 64, [3, 3, 3], seed=1)
    ref = c.delta_ref(False)
    c.d_ids[0], c.d_ids[2] = -1, c.slots
    pool, conv = c.d_pool.clone(), c.d_conv.clone()
    out = torch.full((9, 2, 64), 5.0, dtype=torch.bfloat16, device=DEV)
    c.delta(ops, False, out=out)
    flagged(ops, IndexError)
    assert (out[:3] == 5).all() and (out[6:] == 5).all()
    close(out[3:6], ref[3:6], 2.0 ** -12)
    c.commit(ops, [2, -1, 2])
    flagged(ops, IndexError)
    assert torch.equal(c.d_pool, pool) and torch.equal(c.d_conv, conv)
    ops.conv_gate_tree(c.d_x, c.d_conv[:, 1], c.d_ids, bf(c.w), *c.tree, c.d_b, c.d_a, f32(c.a_log),
                       f32(c.dt))
    flagged(ops, IndexError)


@pytest.mark.parametrize("nodes", [2, 40])
@pytest.mark.parametrize("page", [-1, 10 ** 6, None])
def test_pages_that_are_not_there(ops, page, nodes):  # noqa: F811
    """A page outside the cache, or a sequence longer than its table row: flagged, not
    read, the other sequences as always."""
    ctx, lens = [40, 300, 20], [nodes, nodes, 1]
    c, trees = Paged(1, 128, 16, ctx, lens, 3), R.make_trees(lens, 1)
    q = rnd(np.random.default_rng(0), sum(lens), 2, 128)
    ref, size = R.attention(q, c.ks, c.vs, ctx, trees, 128 ** -0.5)
    table = c.d_table
    if page is None:
        table = table[:, :10].contiguous()
    else:
        table[1, 5] = page
    out = ops.attention_tree(bf(q), c.d_k, c.d_v, table, c.d_ctx, i32(R.cu_of(lens)),
                             i32(np.concatenate(trees)), nodes, c.most)
    flagged(ops, IndexError)
    for r in (0, 2):
        attn_close(out[rows_of(lens, r)], ref[rows_of(lens, r)], size[rows_of(lens, r)])
    pos, slot = ops.tree_slot_map(table, c.d_ctx, i32(R.cu_of(lens)), i32(np.concatenate(trees)), nodes,
                                  16, sum(lens))
    if page is None:
        flagged(ops, IndexError)
        assert (slot[rows_of(lens, 1)] == -1).all()


def test_sequences_longer_than_announced(ops):  # noqa: F811
    ctx, lens = [40, 30], [3, 3]
    c, trees = Paged(1, 64, 16, ctx, lens, 3), R.make_trees(lens, 1)
    q = rnd(np.random.default_rng(0), 6, 2, 64)
    ref, size = R.attention(q, c.ks, c.vs, ctx, trees, 64 ** -0.5)
    for long in (41, -1):
        c.d_ctx[0] = long
        out = torch.full((6, 2, 64), 3.0, dtype=torch.bfloat16, device=DEV)
        ops.attention_tree(bf(q), c.d_k, c.d_v, c.d_table, c.d_ctx, i32([0, 3, 6]),
                           i32(np.concatenate(trees)), 3, 43, out=out)
        flagged(ops, ValueError)
        assert (out[:3] == 3).all(), "skipped"
        attn_close(out[3:], ref[3:], size[3:])


def test_positions_and_slots_outside(ops):  # noqa: F811
    r = np.random.default_rng(0)
    d = bf(rnd(r, 5, 4, 64))
    kc, vc = (torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    cs = f32(np.concatenate([np.ones((10, 16)), np.zeros((10, 16))], 1))
    w = bf(np.ones(64))
    out = torch.full((5, 2, 64), 3.0, dtype=torch.bfloat16, device=DEV)
    call = lambda pos, slot: ops.qk_norm_rope_cache(d[:, :2], d[:, 2:3], d[:, 3:], w, w, cs, i64(pos),
                                                    kc, vc, i32(slot), out=out)
    call([0, 10, -1, 9, 1 << 40], [0, 1, 2, 3, 4])
    flagged(ops, IndexError)
    ref = R.norm_rope(host(d[:, :3]), np.ones(64), np.ones((5, 16)), np.zeros((5, 16)), 1e-6, 0)
    good = [0, 3]
    close(out[good], ref[good][:, :2], 2.0 ** -18)
    assert (out[[1, 2, 4]] == 3).all()
    k = host(kc).reshape(8, 1, 64)
    close(k[[0, 3]], ref[good][:, 2:], 2.0 ** -18)
    assert (k[[1, 2, 4, 5, 6, 7]] == 0).all()
    kc.zero_(), vc.zero_()
    call([0, 1, 2, 3, 4], [8, -2, -1, 7, 1 << 30])
    flagged(ops, IndexError)
    close(out, ref[:, :2], 2.0 ** -18)
    assert (host(kc).reshape(8, 64)[:7] == 0).all() and (host(vc).reshape(8, 64)[:7] == 0).all()
    assert torch.equal(vc.view(8, 64)[7], d[3, 3])


def test_empty_calls(ops):  # noqa: F811
    z = lambda *s, t=torch.bfloat16: torch.zeros(*s, dtype=t, device=DEV)
    i = lambda n: z(n, t=torch.int32)
    pool, conv = z(2, 2, 64, 64, t=torch.float32), z(2, 256, 3)
    for n_seqs in (0, 3):                               # no sequences, or only empty ones
        ids = torch.arange(n_seqs, device=DEV) % 2
        tree = (i(n_seqs + 1), i(0), 4)
        y, g, b = ops.conv_gate_tree(z(0, 256), conv, ids, z(256, 4), *tree, z(0, 2), z(0, 2),
                                     z(2, t=torch.float32), z(2, t=torch.float32))
        assert y.shape == (0, 256) and g.shape == (0, 2)
        args = (z(0, 1, 64), z(0, 2, 64), z(0, 2, t=torch.float32), z(0, 2))
        assert ops.gated_delta_rule_tree(z(0, 1, 64), *args, pool, ids, *tree).shape == (0, 2, 64)
        ops.commit_tree(z(0, 256), *args, conv, pool, ids, *tree, i(n_seqs))
        kc = z(2, 16, 1, 64)
        assert ops.qk_norm_rope_cache(z(0, 2, 64), z(0, 1, 64), z(0, 1, 64), z(64), z(64),
                                      z(4, 16, t=torch.float32), i(0), kc, kc.clone(),
                                      i(0)).shape == (0, 2, 64)
        assert ops.attention_tree(z(0, 2, 64), kc, kc, z(n_seqs, 2, t=torch.int32), i(n_seqs), *tree,
                                  16).shape == (0, 2, 64)
        pos, slot = ops.tree_slot_map(z(n_seqs, 2, t=torch.int32), i(n_seqs), *tree, 16, 0)
        assert pos.shape == (0,) and slot.shape == (0,)
    # rows, but all of them behind the (empty) sequences
    tree = (i(3), i(4), 2)
    out = torch.full((4, 2, 64), 7.0, dtype=torch.bfloat16, device=DEV)
    ops.attention_tree(z(4, 2, 64), kc, kc, z(2, 2, t=torch.int32), i(2), *tree, 16, out=out)
    assert (out == 7).all()
    pos, slot = ops.tree_slot_map(z(2, 2, t=torch.int32), i(2), *tree, 16, 4)
    assert (pos == 0).all() and (slot == -1).all()
    assert ops.check_status() == 0


def test_offsets_past_32_bits(ops):  # noqa: F811
    """A state pool and caches of more than 2^31 elements, used at both ends."""
    c = Gdn(1, 2, 128, [7, 9], seed=6)
    big = torch.empty(70000, 2, 128, 128, device=DEV)   # 2.3e9 floats
    ids = [69999, 0]
    for s, at in zip(c.ids, ids):
        big[at] = c.d_pool[s, 1]
    conv = torch.zeros(70000, c.C, 3, dtype=torch.bfloat16, device=DEV)
    for s, at in zip(c.ids, ids):
        conv[at] = c.d_conv[s, 1]
    out = ops.gated_delta_rule_tree(c.d_q, c.d_k, c.d_v, c.d_g, c.d_beta, big, i64(ids), *c.tree)
    close(out, c.delta_ref(False), 2.0 ** -12)
    ops.commit_tree(c.d_x, c.d_k, c.d_v, c.d_g, c.d_beta, conv, big, i64(ids), *c.tree, i32([5, 8]))
    win, st = c.commit_ref([5, 8])
    for r, at in enumerate(ids):
        assert np.linalg.norm(host(big[at]) - st[r]) <= 1e-5 * np.linalg.norm(st[r])
        assert np.array_equal(host(conv[at]), win[r])
    del big, conv
    block, blocks = 256, 20000                          # 20000 x 256 x 4 x 128 = 2.6e9
    kc = torch.empty(blocks, block, 4, 128, dtype=torch.bfloat16, device=DEV)
    vc = torch.empty_like(kc)
    p, trees = Paged(4, 128, 256, [300, 10], [5, 20], 4), R.make_trees([5, 20], 4)
    where = np.array([19999, 3, 19998])
    used = [p.table[0, 0], p.table[0, 1], p.table[1, 0]]
    for a, b in zip(where, used):
        kc[a], vc[a] = p.d_k[b], p.d_v[b]
    table = i32([[19999, 3, -1], [19998, -1, -1]])
    q = rnd(np.random.default_rng(2), 25, 8, 128)
    out = ops.attention_tree(bf(q), kc, vc, table, i32([300, 10]), i32([0, 5, 25]),
                             i32(np.concatenate(trees)), 20, 305)
    ref, size = R.attention(q, p.ks, p.vs, [300, 10], trees, 128 ** -0.5)
    attn_close(out, ref, size)
    d = bf(rnd(np.random.default_rng(1), 2, 9, 128))
    cs, w = f32(np.concatenate([np.ones((4, 64)), np.zeros((4, 64))], 1)), bf(np.ones(128))
    slots = [19999 * 256 + 255, 19998 * 256]
    ops.qk_norm_rope_cache(d[:, :1], d[:, 1:5], d[:, 5:], w, w, cs, i64([0, 1]), kc, vc, i32(slots))
    assert torch.equal(vc[19999, 255], d[0, 5:]) and torch.equal(vc[19998, 0], d[1, 5:])
    assert ops.check_status() == 0
