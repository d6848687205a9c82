"""The tree operators as a program uses them: many sequences, odd head groups, views of
fused projections, captured and replayed, two streams at once, the same bits again."""
import numpy as np
import pytest
import torch

import _tree_reference as R
from test_gpu_tree import DEV, Gdn, Paged, attn_close, bf, f32, host, i32, i64, ops, rnd  # noqa: F401
from test_gpu_tree_faults import flagged, rows_of

pytestmark = pytest.mark.gpu


def attend(ops, c, q, lens, trees, out=None):  # noqa: F811
    par = np.concatenate(list(trees) + [np.full(q.shape[0] - sum(lens), -7)])
    return ops.attention_tree(q, c.d_k, c.d_v, c.d_table, c.d_ctx, i32(R.cu_of(lens)), i32(par),
                              max(lens), c.most, out=out)


@pytest.mark.parametrize("HQ,HKV,D,lens", [
    (3, 1, 128, [50, 3, 42, 43]),       # 42 whole nodes of three heads to a row tile
    (10, 2, 64, [26, 25, 64]),          # 25 of five
    (12, 1, 128, [64, 10, 11]),
    (128, 1, 64, [3, 1]),               # one node a tile
    (130, 1, 64, [2, 1]),               # less than one
    (65, 1, 128, [2, 5]),
    (20, 1, 256, [4, 13]),
])
def test_attention_head_groups(ops, HQ, HKV, D, lens):  # noqa: F811
    ctx = [130, 64, 7, 0][:len(lens)]
    c, trees = Paged(HKV, D, 16, ctx, lens, 5), R.make_trees(lens, 5)
    q = rnd(np.random.default_rng(1), sum(lens), HQ, D)
    ref, size = R.attention(q, c.ks, c.vs, ctx, trees, D ** -0.5)
    attn_close(attend(ops, c, bf(q), lens, trees), ref, size)
    assert ops.check_status() == 0


@pytest.mark.parametrize("D,most,HQ", [(128, 1, 2), (128, 12, 4), (64, 6, 8), (64, 3, 2), (256, 9, 4)])
def test_attention_many_sequences(ops, D, most, HQ):  # noqa: F811
    """More sequences than threads that scan their lengths, empty ones among them, several
    units to a CTA and CTAs that begin in the middle of one."""
    r = np.random.default_rng(D + most)
    lens, ctx = r.integers(0, most + 1, 410).tolist(), r.integers(0, 150, 410).tolist()
    lens[0], lens[380:390], lens[409], ctx[200] = 0, [0] * 10, most, 900
    c, trees = Paged(1, D, 64, ctx, lens, 8), R.make_trees(lens, 8)
    q = rnd(r, sum(lens), HQ, D)
    ref, size = R.attention(q, c.ks, c.vs, ctx, trees, D ** -0.5)
    got = attend(ops, c, bf(q), lens, trees)
    attn_close(got, ref, size)
    assert torch.equal(got, attend(ops, c, bf(q), lens, trees)), "the same bits again"
    assert ops.check_status() == 0


@pytest.mark.parametrize("nodes", [6, 20])
def test_attention_malformed_parents(ops, nodes):  # noqa: F811
    ctx, lens = [40, 300, 20], [nodes] * 3
    c, trees = Paged(1, 128, 16, ctx, lens, 3), R.make_trees(lens, 1)
    q = rnd(np.random.default_rng(0), sum(lens), 4, 128)
    ref, size = R.attention(q, c.ks, c.vs, ctx, trees, 128 ** -0.5)
    for parent in (4, 1 << 30, -2):
        bad = [t.copy() for t in trees]
        bad[1][4] = parent
        out = attend(ops, c, bf(q), lens, bad)
        flagged(ops, ValueError)
        for r in (0, 2):
            attn_close(out[rows_of(lens, r)], ref[rows_of(lens, r)], size[rows_of(lens, r)])


@pytest.mark.parametrize("nodes,D", [(3, 128), (20, 128), (10, 64), (5, 256)])
def test_attention_views_and_rows_behind(ops, nodes, D):  # noqa: F811
    """Queries and caches as views of wider tensors; rows behind the last sequence stay."""
    ctx, lens = [70, 5], [nodes, 2]
    c, trees = Paged(2, D, 16, ctx, lens, 3), R.make_trees(lens, 1)
    n, r = sum(lens), np.random.default_rng(0)
    q = rnd(r, n, 4, D)
    wide = torch.full((n + 3, 6 * D), float("nan"), dtype=torch.bfloat16, device=DEV)
    wide[:n, D:5 * D] = bf(q).view(n, -1)
    both = torch.full((*c.d_k.shape[:2], 3, 2, D), float("nan"), dtype=torch.bfloat16, device=DEV)
    both[:, :, 1], both[:, :, 2] = c.d_k, c.d_v
    c.d_k, c.d_v = both[:, :, 1], both[:, :, 2]
    out = torch.full((n + 3, 4, D), 7.0, dtype=torch.bfloat16, device=DEV)
    attend(ops, c, wide[:, D:5 * D].view(n + 3, 4, D), lens, trees, out=out)
    ref, size = R.attention(q, c.ks, c.vs, ctx, trees, D ** -0.5)
    attn_close(out[:n], ref, size)
    assert (out[n:] == 7).all()


class Step:
    """All six operators over one batch, on fixed buffers."""

    def __init__(self, ops, lens, seed, HQ=4, HKV=2):  # noqa: F811
        self.ops, self.lens = ops, lens
        self.g = Gdn(2, 4, 128, lens, seed=seed)
        ctx = [17 * (i + 1) % 90 for i in range(len(lens))]
        self.c = Paged(HKV, 128, 16, ctx, lens, seed)
        r = np.random.default_rng(seed)
        self.qkv = bf(rnd(r, self.g.N, HQ + 2 * HKV, 128))
        self.w = bf(rnd(r, 2, 128))
        self.cs = f32(rnd(r, 300, 64))
        self.HQ, self.HKV = HQ, HKV
        self.acc = i32([m - 1 if m else -1 for m in lens])

    def run(self):
        ops, g, c, q = self.ops, self.g, self.c, self.qkv  # noqa: F811
        y, gate, beta = ops.conv_gate_tree(g.d_x, g.d_conv[:, 1], g.d_ids, bf_w(g), *g.tree, g.d_b, g.d_a,
                                           g.f_log, g.f_dt)
        hk = g.d_k.shape[1] * 128
        rows = y.shape[0]
        yq, yk, yv = (t.view(rows, -1, 128) for t in y.split([hk, hk, y.shape[1] - 2 * hk], 1))
        o = ops.gated_delta_rule_tree(yq, yk, yv, gate, beta, g.d_pool[:, 1], g.d_ids, *g.tree)
        pos, slot = ops.tree_slot_map(c.d_table, c.d_ctx, *g.tree, 16, rows)
        qn = ops.qk_norm_rope_cache(q[:, :self.HQ], q[:, self.HQ:self.HQ + self.HKV],
                                    q[:, self.HQ + self.HKV:], self.w[0], self.w[1], self.cs, pos,
                                    c.d_k, c.d_v, slot)
        a = ops.attention_tree(qn, c.d_k, c.d_v, c.d_table, c.d_ctx, *g.tree, 200)
        ops.commit_tree(g.d_x, yk, yv, gate, beta, g.d_conv[:, 1], g.d_pool[:, 1], g.d_ids, *g.tree,
                        self.acc)
        n = sum(self.lens)
        return o[:n], a[:n], pos, slot

    def state(self):
        return [t.clone() for t in (self.g.d_conv, self.g.d_pool, self.c.d_k, self.c.d_v)]


def bf_w(g):
    if not hasattr(g, "b_w"):
        g.b_w, g.f_log, g.f_dt = bf(g.w), f32(g.a_log), f32(g.dt)
    return g.b_w


def same(a, b):
    return all(torch.equal(x.nan_to_num(5), y.nan_to_num(5)) for x, y in zip(a, b))


LENS = [5, 0, 33, 1, 12]


def test_a_captured_step_replays_with_new_contents(ops):  # noqa: F811
    """Captured once, replayed after every input has changed in place: what eager calls
    give, bit for bit."""
    one, two = Step(ops, LENS, 1), Step(ops, LENS, 2)
    bf_w(one.g), bf_w(two.g)
    fresh = two.state()
    want = [t.clone() for t in two.run()]
    end = two.state()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        one.run()
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = one.run()
    for a, b in ((one.g, two.g), (one.c, two.c), (one, two)):
        for name, t in vars(a).items():
            if isinstance(t, torch.Tensor):
                t.copy_(getattr(b, name))
    for a, b in zip((one.g.d_conv, one.g.d_pool, one.c.d_k, one.c.d_v), fresh):
        a.copy_(b)
    graph.replay()
    torch.cuda.synchronize()
    assert same(got, want) and same(one.state(), end)
    for a, b in zip((one.g.d_conv, one.g.d_pool, one.c.d_k, one.c.d_v), fresh):
        a.copy_(b)
    graph.replay()
    torch.cuda.synchronize()
    assert same(got, want) and same(one.state(), end), "and again"
    assert ops.check_status() == 0


def test_two_streams_at_once(ops):  # noqa: F811
    steps = [Step(ops, LENS, 3), Step(ops, [40, 2, 0, 64], 4)]
    fresh = [s.state() for s in steps]
    want = []
    for s in steps:
        bf_w(s.g)
        want.append([t.clone() for t in s.run()])
    ends = [s.state() for s in steps]
    streams = [torch.cuda.Stream() for _ in steps]
    for _ in range(5):
        for s, f in zip(steps, fresh):
            for a, b in zip((s.g.d_conv, s.g.d_pool, s.c.d_k, s.c.d_v), f):
                a.copy_(b)
        torch.cuda.synchronize()
        got = []
        for s, st in zip(steps, streams):
            with torch.cuda.stream(st):
                got.append(s.run())
        torch.cuda.synchronize()
        for s, g, w, e in zip(steps, got, want, ends):
            assert same(g, w) and same(s.state(), e)
    assert ops.check_status() == 0


def test_a_slot_named_twice_is_read_twice(ops):  # noqa: F811
    """Reading operators: two sequences may start from one stored state (a prefix that two
    requests share)."""
    c = Gdn(1, 2, 128, [6, 6], seed=2)
    alone = c.delta(ops, False)
    c.d_ids[1] = c.d_ids[0]
    both = c.delta(ops, False)
    assert torch.equal(both[:6], alone[:6])
    c.d_ids[0] = c.d_ids[1] = c.ids[1]
    assert torch.equal(c.delta(ops, False)[6:], alone[6:])
    ops.set_debug_checks(True)                          # (they let the pool's last slot be named twice)
    try:
        c.d_ids[:] = 0
        c.delta(ops, False)
        with pytest.raises(ValueError, match="appears 2 times"):
            c.commit(ops, [1, 1])
        c.d_ids[1] = -1
        with pytest.raises(IndexError):
            c.delta(ops, False)
    finally:
        ops.set_debug_checks(False)


@pytest.mark.parametrize("D,HQ", [(128, 2), (128, 8), (64, 2), (256, 4)])
@pytest.mark.parametrize("most", [64, 65, 128, 129])
def test_attention_within_one_tile(ops, D, HQ, most):  # noqa: F811
    """Bounds around one tile of positions, where no joining launch follows."""
    ctx, lens = [most - 9, 0, 30, 11], [9, 1, 0, 6]
    c, trees = Paged(1, D, 32, ctx, lens, most), R.make_trees(lens, 5)
    assert c.most == most
    q = rnd(np.random.default_rng(most), sum(lens), HQ, D)
    ref, size = R.attention(q, c.ks, c.vs, ctx, trees, D ** -0.5)
    attn_close(attend(ops, c, bf(q), lens, trees), ref, size)
    assert ops.check_status() == 0
