"""The tree operators together, as a server uses them: the drop-in layer checks a
drafted tree and takes the accepted path over, against the same layer decoding the
path's tokens one by one; the attention side from slot map to the compacted cache;
and everything captured into CUDA graphs.

Tolerances: the layer's projections are library GEMMs whose results differ by bf16
roundings between batch sizes, hence the layer tests' output max-abs 2e-2 and state
relative 2e-2; conv windows hold projection rows and get the outputs' tolerance.
"""
import types

import numpy as np
import pytest
import torch

import _tree_reference as R
from test_gpu_tree import U, bf, f32, host, i32, i64, rnd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def pkg_gpu(pkg):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.set_device(0)
    return pkg


def make_layer(pkg, D, HK=2, HV=4, hidden=256, seed=0):
    cfg = types.SimpleNamespace(hidden_size=hidden, linear_num_key_heads=HK,
                                linear_num_value_heads=HV, linear_key_head_dim=D,
                                linear_value_head_dim=D, linear_conv_kernel_dim=4,
                                rms_norm_eps=1e-6)
    prev = torch.get_default_dtype()
    torch.set_default_dtype(torch.bfloat16)
    try:
        with torch.device(DEV), torch.no_grad():
            m = pkg.layer.Qwen3_5GatedDeltaNet(cfg)
            g = torch.Generator(device=DEV).manual_seed(seed)
            m._fused_weight().normal_(0, hidden ** -0.5, generator=g)
            m.conv1d.weight.uniform_(-0.5, 0.5, generator=g)
            m.A_log.uniform_(-1.0, 0.0, generator=g)
            m.dt_bias.zero_()
            m.out_proj.weight.normal_(0, (HV * D) ** -0.5, generator=g)
    finally:
        torch.set_default_dtype(prev)
    return m


def forward(pkg, m, x, ids, lens, parents=None):
    cu = i32(R.cu_of(lens))
    if parents is None:
        pkg.context.set_context(cu, cu, max(lens), max(lens), linear_state_ids=ids,
                                lens_q=list(lens))
    else:
        pkg.context.set_draft_context(cu, parents, max(lens), ids)
    try:
        with torch.inference_mode():
            return m(None, x)
    finally:
        pkg.context.reset_context()


@pytest.mark.parametrize("D", [128, 64])
def test_layer_checks_a_tree_and_commits(pkg_gpu, D):
    pkg = pkg_gpu
    m = make_layer(pkg, D)
    pools = pkg.state_pool.StatePools([m], 6, DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    lens, prompt = [7, 1, 12], [40, 9, 70]
    ids = i64([4, 0, 2])
    rows = lambda n: torch.randn(n, 256, generator=g, device=DEV).to(torch.bfloat16)
    forward(pkg, m, rows(sum(prompt)), ids, prompt)
    s0, c0 = pools.s_pool.clone(), pools.conv_pool.clone()
    trees = R.make_trees(lens, 3)
    x = rows(sum(lens))
    y = forward(pkg, m, x, ids, lens, i32(np.concatenate(trees)))
    assert torch.equal(pools.s_pool, s0) and torch.equal(pools.conv_pool, c0), "checked, not taken"
    accepted = [6, -1, 9]
    m.commit_drafts(i32(accepted))
    with pytest.raises(RuntimeError, match="once"):
        m.commit_drafts(i32(accepted))
    s1, c1 = pools.s_pool.clone(), pools.conv_pool.clone()
    nxt = rows(3)
    y1 = forward(pkg, m, nxt, ids, [1, 1, 1])
    # the same tokens one by one
    at = 0
    for r, par in enumerate(trees):
        for node in {accepted[r], len(par) - 1} - {-1}:
            pools.s_pool.copy_(s0)
            pools.conv_pool.copy_(c0)
            for i in R.ancestors(par, node):
                o = forward(pkg, m, x[at + i:at + i + 1], ids[r:r + 1], [1])
                assert (o - y[at + i]).abs().max() <= 2e-2
            if node == accepted[r]:
                s = int(ids[r])
                assert (pools.s_pool[s] - s1[s]).norm() <= 2e-2 * s1[s].norm()
                assert (pools.conv_pool[s].float() - c1[s].float()).abs().max() <= 2e-2
                o = forward(pkg, m, nxt[r:r + 1], ids[r:r + 1], [1])
                assert (o - y1[r]).abs().max() <= 3e-2
        at += len(par)
    assert torch.equal(s1[0], s0[0]), "nothing accepted: the slot keeps its state"
    assert pkg.ops.check_status() == 0


def attention_side(ops, row, qw, kw, cs, kc, vc, table, ctx, cu, par, most, HQ, HKV, D, acc):
    """One round of an attention layer: slots, norms + rotation + store, attention, and
    the accepted rows stored where they belong."""
    n, block = row.shape[0], kc.shape[1]
    d = row.view(n, HQ + 2 * HKV, D)
    parts = (d[:, :HQ], d[:, HQ:HQ + HKV], d[:, HQ + HKV:])
    pos, slot = ops.tree_slot_map(table, ctx, cu, par, 64, block, n)
    q = ops.qk_norm_rope_cache(*parts, qw, kw, cs, pos, kc, vc, slot, unit_offset=True)
    o = ops.attention_tree(q, kc, vc, table, ctx, cu, par, 64, most)
    _, kept = ops.tree_slot_map(table, ctx, cu, par, 64, block, n, accepted=acc)
    ops.qk_norm_rope_cache(*parts, qw, kw, cs, pos, kc, vc, kept, unit_offset=True)
    return pos, q, o


def test_attention_side_compacts_the_accepted_path(pkg_gpu):
    ops = pkg_gpu.ops
    r = np.random.default_rng(5)
    HQ, HKV, D, block, rot = 4, 2, 64, 16, 32
    lens, ctx, accepted = [9, 20, 3], [30, 0, 47], [7, 15, -1]
    n, trees = sum(lens), R.make_trees(lens, 8)
    row, qw, kw = rnd(r, n, (HQ + 2 * HKV) * D), rnd(r, D, std=0.1), rnd(r, D, std=0.1)
    ang = np.arange(200)[:, None] * 10.0 ** (-np.arange(rot // 2) / 8)
    cs = np.concatenate([np.cos(ang), np.sin(ang)], 1).astype(np.float32)
    table = r.permutation(30).reshape(3, 10)[:, :6]
    kc, vc = bf(rnd(r, 30, block, HKV, D)), bf(rnd(r, 30, block, HKV, D))
    k0, v0 = kc.clone(), vc.clone()
    args = (bf(row), bf(qw), bf(kw), f32(cs), kc, vc, i32(table))
    tail = (i32(R.cu_of(lens)), i32(np.concatenate(trees)), 100, HQ, HKV, D, i32(accepted))
    pos, q, o = attention_side(ops, *args, i32(ctx), *tail)
    # in 64 bits, from the rotated rows the kernel itself rounded
    at = lambda c, s, p: host(c)[table[s][p // block], p % block]
    x = row.reshape(n, -1, D)
    c, s = (t.astype(np.float64) for t in np.split(cs[pos.cpu().numpy()], 2, 1))
    kr = bf(R.norm_rope(x[:, HQ:HQ + HKV], kw, c, s, 1e-6, 1.0))
    ks, vs, start = [], [], 0
    for i, m in enumerate(lens):
        p = np.arange(ctx[i])
        ks.append(np.concatenate([at(k0, i, p), host(kr)[start:start + m]]))
        vs.append(np.concatenate([at(v0, i, p), x[start:start + m, HQ + HKV:]]))
        start += m
    ref, size = R.attention(host(q), ks, vs, ctx, trees, D ** -0.5)
    # the keys' rounding may fall to the other side here and there: scores differ by u |q| |k|
    assert (np.abs(host(o) - ref) <= U * np.abs(ref) + 3 * U * size + 1e-3).all()
    start = 0
    for i, m in enumerate(lens):
        path = R.ancestors(trees[i], accepted[i])
        p = ctx[i] + np.arange(len(path))
        if path:
            assert np.array_equal(at(vc, i, p), x[start + np.array(path), HQ + HKV:])
            assert (np.abs(at(kc, i, p) - host(kr)[start + np.array(path)]) <= 2 * U * np.abs(
                host(kr)[start + np.array(path)]) + 1e-6).all()
        p = np.arange(ctx[i])
        assert np.array_equal(at(kc, i, p), at(k0, i, p)), "the context stays"
        start += m
    assert ops.check_status() == 0


def test_everything_in_graphs_on_two_streams(pkg_gpu):
    """A layer's check and commit and an attention round, captured; replayed with other
    inputs, two graphs at once on two streams, they give what eager calls give."""
    pkg, ops = pkg_gpu, pkg_gpu.ops
    lens, HQ, HKV, D = [5, 8, 1, 0, 3], 4, 1, 128
    n, trees = sum(lens), R.make_trees(lens, 2)
    r = np.random.default_rng(1)
    cu, par = i32(R.cu_of(lens)), i32(np.concatenate(trees))
    acc = i32([4, 3, 0, -1, 1])
    table, ctx = i32(r.permutation(5 * 40).reshape(5, 40)), i32([600, 37, 0, 5, 255])
    cs = f32(r.standard_normal((700, 64)))
    ids = i64([3, 1, 0, 5, 2])

    class World:
        def __init__(self, seed):
            self.m = make_layer(pkg, 64, seed=seed)
            self.pools = pkg.state_pool.StatePools([self.m], 6, DEV)
            g = torch.Generator(device=DEV).manual_seed(seed)
            self.x = torch.randn(n, 256, generator=g, device=DEV).to(torch.bfloat16)
            self.row = torch.randn(n, (HQ + 2 * HKV) * D, generator=g, device=DEV).to(torch.bfloat16)
            self.w = torch.randn(D, generator=g, device=DEV).to(torch.bfloat16)
            self.kc = torch.randn(200, 16, HKV, D, generator=g, device=DEV).to(torch.bfloat16)
            self.vc = torch.randn(200, 16, HKV, D, generator=g, device=DEV).to(torch.bfloat16)
            self.pools.s_pool.normal_(0, 0.1, generator=g)
            self.pools.conv_pool.normal_(0, 1, generator=g)

        def state(self):
            return [self.pools.s_pool, self.pools.conv_pool, self.kc, self.vc]

        def run(self):
            y = forward_in(self)
            self.m.commit_drafts(acc)
            self.out = [y, attention_side(ops, self.row, self.w, self.w, cs, self.kc, self.vc, table,
                                          ctx, cu, par, 700, HQ, HKV, D, acc)[2]]
            return self.out

    def forward_in(world):
        pkg.context.set_draft_context(cu, par, 8, ids)
        with torch.inference_mode():
            return world.m(None, world.x)

    worlds = [World(1), World(2)]
    graphs, streams = [], [torch.cuda.Stream() for _ in worlds]
    for w, st in zip(worlds, streams):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            keep = [t.clone() for t in w.state()]
            w.run()
            for t, k in zip(w.state(), keep):
                t.copy_(k)
            torch.cuda.synchronize()
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=st):
                w.run()
            graphs.append(gr)
    torch.cuda.synchronize()
    captured = [w.out for w in worlds]
    for w, seed in zip(worlds, (7, 8)):
        g = torch.Generator(device=DEV).manual_seed(seed)
        w.x.normal_(generator=g)
        w.row.normal_(generator=g)
    keep = [[t.clone() for t in w.state()] for w in worlds]
    torch.cuda.synchronize()
    for gr, st in zip(graphs, streams):
        with torch.cuda.stream(st):
            gr.replay()
    torch.cuda.synchronize()
    got = [[t.clone() for t in c + w.state()] for c, w in zip(captured, worlds)]
    for w, k, mine in zip(worlds, keep, got):
        for t, old in zip(w.state(), k):
            t.copy_(old)
        again = w.run() + w.state()
        torch.cuda.synchronize()
        for a, b in zip(again, mine):
            assert torch.equal(a, b)
    pkg.context.reset_context()
    assert ops.check_status() == 0
