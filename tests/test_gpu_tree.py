"""The operators for trees of drafted tokens against 64-bit restatements.

Tolerances (u = 2^-8, half a bf16 step relative to the value):
* conv output, rotated queries and keys, delta rule: one rounding, u |ref|, plus
  what fp32 sums and 16-bit operand pairs leave of the row's largest value
  (2^-12 of it for the delta rule: two operands of 2^-17 each in sums of up to 192
  terms; 2^-18 for the others);
* attention: the probabilities are rounded to bf16 for the second product, at
  most u of each, so u sum(p |v|), and the output's own rounding;
* committed states: each of a path's tokens adds a few fp32 roundings, taken as
  2^-24 (8 depth + 32) of the state's norm;
* whole numbers, copies, windows and what must stay untouched: exact.
"""
import numpy as np
import pytest
import torch

import _tree_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -8


@pytest.fixture(scope="module")
def ops(pkg):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.set_device(0)
    return pkg.ops


def rnd(r, *shape, std=1.0):
    """bf16-representable normal values."""
    t = torch.from_numpy((r.standard_normal(shape) * std).astype(np.float32))
    return t.to(torch.bfloat16).double().numpy()


def bf(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(DEV).to(torch.bfloat16)


def f32(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(DEV)


def i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(DEV)


def i64(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int64)).to(DEV)


def host(t):
    return t.double().cpu().numpy()


def close(got, ref, slack, what=""):
    """|got - ref| <= u |ref| + slack of the row's largest value."""
    got = host(got) if isinstance(got, torch.Tensor) else got
    tol = U * np.abs(ref) + slack * np.abs(ref).max(-1, keepdims=True) + 1e-30
    bad = ~(np.abs(got - ref) <= tol)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size}, worst " \
        f"{np.nanmax(np.abs(got - ref) / tol):.2f} of the tolerance, NaN {np.isnan(got).sum()}"


# ---------------------------------------------------------------------------
# the GDN side
# ---------------------------------------------------------------------------


class Gdn:
    """One layer's inputs: rows are column views of a projection, pools hold two layers."""

    def __init__(self, HK, HV, D, lens, seed, K=4, chain=False, wide=4, pad_rows=0):
        r = np.random.default_rng(seed)
        self.HK, self.HV, self.D, self.K, self.lens = HK, HV, D, K, lens
        self.n, self.C = sum(lens), (2 * HK + HV) * D
        n, C = self.n + pad_rows, self.C
        self.N = n
        self.trees = R.make_trees(lens, seed, chain, wide)
        self.slots = len(lens) + 3
        self.ids = r.permutation(self.slots)[:len(lens)]
        self.row = rnd(r, n, C + HV * D + 2 * HV + 8)
        self.x, self.z = self.row[:, :C], self.row[:, C:C + HV * D].reshape(n, HV, D)
        self.b, self.a = self.row[:, C + HV * D:][:, :HV], self.row[:, C + HV * D + HV:][:, :HV]
        self.w = rnd(r, C, K, std=0.3)
        self.a_log, self.dt = r.uniform(-1, 1, HV).astype(np.float32), r.uniform(-.5, .5, HV).astype(np.float32)
        self.y = rnd(r, n, C)
        self.g = -np.log1p(np.exp(r.standard_normal((n, HV)))).astype(np.float32)
        self.beta = rnd(r, n, HV) * 0 + torch.sigmoid(torch.from_numpy(rnd(r, n, HV))).to(torch.bfloat16).double().numpy()
        self.nw = 1 + rnd(r, D, std=0.125)
        self.nw = bf(self.nw).double().cpu().numpy()
        self.conv = rnd(r, self.slots, 2, C, K - 1)
        self.pool = (r.standard_normal((self.slots, 2, HV, D, D)) * 0.3).astype(np.float32)
        self.upload()

    def upload(self):
        C, HV, D, HK, n = self.C, self.HV, self.D, self.HK, self.N
        self.d_row = bf(self.row)
        self.d_x, self.d_z = self.d_row[:, :C], self.d_row[:, C:C + HV * D].view(n, HV, D)
        self.d_b, self.d_a = self.d_row[:, C + HV * D:][:, :HV], self.d_row[:, C + HV * D + HV:][:, :HV]
        y = bf(self.y)
        self.d_q, self.d_k = y[:, :HK * D].view(n, HK, D), y[:, HK * D:2 * HK * D].view(n, HK, D)
        self.d_v = y[:, 2 * HK * D:].view(n, HV, D)
        self.d_g, self.d_beta = f32(self.g), bf(self.beta)
        self.d_conv, self.d_pool = bf(self.conv), f32(self.pool)
        self.d_cu = i32(R.cu_of(self.lens))
        par = np.concatenate(self.trees + [np.full(self.N - self.n, -7)])   # pad rows hold rubbish
        self.d_par, self.d_ids = i32(par), i64(self.ids)
        self.tree = (self.d_cu, self.d_par, max(max(self.lens), 1))

    def qkv(self):
        kd = self.HK * self.D
        y = self.y[:self.n]
        return (y[:, :kd].reshape(-1, self.HK, self.D), y[:, kd:2 * kd].reshape(-1, self.HK, self.D),
                y[:, 2 * kd:].reshape(-1, self.HV, self.D))

    def delta(self, ops, norm, **kw):
        kw = dict(z=self.d_z, norm_weight=bf(self.nw), eps=1e-6, **kw) if norm else kw
        return ops.gated_delta_rule_tree(self.d_q, self.d_k, self.d_v, self.d_g, self.d_beta,
                                         self.d_pool[:, 1], self.d_ids, *self.tree, **kw)

    def delta_ref(self, norm):
        q, k, v = self.qkv()
        n = self.n
        return R.delta(q, k, v, self.g[:n].astype(np.float64), self.beta[:n],
                       self.pool[self.ids, 1].astype(np.float64), self.trees,
                       self.z[:n] if norm else None, self.nw)

    def commit(self, ops, accepted):
        ops.commit_tree(self.d_x, self.d_k, self.d_v, self.d_g, self.d_beta, self.d_conv[:, 1],
                        self.d_pool[:, 1], self.d_ids, *self.tree, i32(accepted))

    def commit_ref(self, accepted):
        q, k, v = self.qkv()
        n = self.n
        return R.commit(self.x[:n], k, v, self.g[:n].astype(np.float64), self.beta[:n],
                        self.conv[self.ids, 1], self.pool[self.ids, 1].astype(np.float64),
                        self.trees, accepted)

    def check_pools(self, accepted, what=""):
        win, st = self.commit_ref(accepted)
        conv, pool = self.conv.copy(), self.pool.astype(np.float64)
        conv[self.ids, 1] = win
        assert np.array_equal(host(self.d_conv), conv), f"{what}: conv windows"
        got = host(self.d_pool)
        for r, s in enumerate(self.ids):
            depth = len(R.ancestors(self.trees[r], accepted[r]))
            err = np.linalg.norm(got[s, 1] - st[r])
            assert err <= 2.0 ** -24 * (8 * depth + 32) * np.linalg.norm(st[r]), f"{what}: seq {r}"
            if depth == 0:
                assert np.array_equal(got[s, 1], pool[s, 1])
        rest = np.setdiff1d(np.arange(self.slots), self.ids)
        assert np.array_equal(got[rest], pool[rest]) and np.array_equal(got[:, 0], pool[:, 0])


DELTA = [
    # HK, HV, D, nodes of the sequences, chain
    (2, 4, 128, [1, 5, 8], False),
    (2, 4, 128, [1, 1, 1, 1], True),
    (1, 4, 64, [3, 0, 16, 9], False),
    (4, 4, 128, [17, 32, 0, 1], False),
    (3, 6, 64, [31, 2], True),
    (1, 2, 128, [64, 33, 48, 1], False),
    (1, 1, 64, [64, 63], True),
    (2, 8, 128, [16, 15, 10], True),
]


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("HK,HV,D,lens,chain", DELTA)
def test_delta_rule(ops, HK, HV, D, lens, chain, norm):
    c = Gdn(HK, HV, D, lens, seed=sum(lens) + D, chain=chain)
    out = c.delta(ops, norm)
    assert np.array_equal(host(c.d_pool), c.pool.astype(np.float64)), "the states are only read"
    close(out, c.delta_ref(norm), 2.0 ** -12)
    assert ops.check_status() == 0


@pytest.mark.parametrize("HK,HV,D,nodes", [(2, 8, 128, 8), (2, 4, 64, 8), (2, 4, 128, 13),
                                          (1, 3, 64, 16), (1, 3, 128, 30), (2, 2, 64, 64),
                                          (1, 2, 128, 40)])
def test_delta_rule_many_units(ops, HK, HV, D, nodes):
    """Many units per CTA, so every buffer is used again and again; empty sequences and
    a slot that is not one among them."""
    r = np.random.default_rng(D + nodes)
    lens = [int(x) for x in r.integers(0, nodes + 1, 150)]
    lens[0], lens[7], lens[8], lens[20] = nodes, 0, 0, 3
    c = Gdn(HK, HV, D, lens, seed=nodes)
    out = torch.zeros(c.N, HV, D, dtype=torch.bfloat16, device=DEV)
    ids = c.d_ids.clone()
    c.d_ids[20] = c.slots
    c.delta(ops, True, out=out)
    with pytest.raises(IndexError):
        ops.check_status()
    start = sum(lens[:20])
    assert (out[start:start + 3] == 0).all()
    c.d_ids = ids
    close(c.delta(ops, True), c.delta_ref(True), 2.0 ** -12)
    again = c.delta(ops, True)
    assert torch.equal(again, c.delta(ops, True)) and ops.check_status() == 0


@pytest.mark.parametrize("D", [128, 64])
def test_delta_rule_extreme_gates(ops, D):
    """No decay, total decay (-inf and far below exp's range), write strengths 0 and 1."""
    c = Gdn(1, 2, D, [12, 40], seed=5)
    c.g[:, 0] = 0.0
    c.g[::3, 1] = -np.inf
    c.g[1::3, 1] = -500.0
    c.beta[::2] = 0.0
    c.beta[1::2] = 1.0
    c.upload()
    close(c.delta(ops, False), c.delta_ref(False), 2.0 ** -12)
    acc = [11, 37]
    c.commit(ops, acc)
    c.check_pools(acc)


def test_delta_rule_equals_single_steps(ops):
    """A chain's rows are the single-step operator's outputs, its commit their state."""
    c = Gdn(2, 4, 128, [6, 6, 6], seed=9, chain=True)
    tree = c.delta(ops, False)
    pool = c.d_pool.clone()
    for i in range(6):
        rows = [i, 6 + i, 12 + i]
        o = ops.recurrent_gdn_inplace(c.d_q[rows], c.d_k[rows], c.d_v[rows], c.d_g[rows],
                                      c.d_beta[rows], pool[:, 1], c.d_ids)
        close(tree[rows], host(o)[:, 0], 2.0 ** -12 + U, f"step {i}")
    c.commit(ops, [5, 5, 5])
    err = (c.d_pool - pool).norm() / pool.norm()
    assert err <= 2.0 ** -24 * (16 * 6 + 64)


@pytest.mark.parametrize("n", [7, 30, 64])
@pytest.mark.parametrize("what", ["k", "v", "q", "g", "beta"])
def test_delta_rule_nan_stays_on_its_path(ops, what, n):
    c = Gdn(1, 2, 128, [n, 3], seed=n, wide=3)
    ref = c.delta_ref(False)
    node = 2
    t = {"k": c.d_k, "v": c.d_v, "q": c.d_q, "g": c.d_g, "beta": c.d_beta}[what]
    t[node].fill_(float("inf") if what == "v" else float("nan"))
    got = host(c.delta(ops, False))
    hit = np.array([node in R.ancestors(c.trees[0], i) for i in range(n)] + [False] * 3)
    if what == "q":
        hit[:] = False
        hit[node] = True
    assert not np.isfinite(got[hit]).any()
    close(got[~hit], ref[~hit], 2.0 ** -12)


def test_delta_rule_rows_and_strides(ops):
    """Unaligned rows (an odd element offset), a single row, and rows behind the last sequence."""
    c = Gdn(2, 4, 128, [4, 3], seed=3, pad_rows=5)
    for t in ("d_q", "d_k", "d_v", "d_z"):
        a = getattr(c, t)
        wide = torch.zeros(c.N, a.shape[1] * a.shape[2] + 3, dtype=torch.bfloat16, device=DEV)
        wide[:, 1:1 + a.shape[1] * a.shape[2]] = a.reshape(c.N, -1)
        setattr(c, t, wide[:, 1:1 + a.shape[1] * a.shape[2]].unflatten(1, a.shape[1:]))
    out = torch.full((c.N, 4, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    got = c.delta(ops, True, out=out)
    assert got is out and (out[c.n:] == 7.0).all(), "rows behind the last sequence"
    close(out[:c.n], c.delta_ref(True), 2.0 ** -12)
    pool = c.d_pool.clone()
    c.commit(ops, [3, -1])
    c.check_pools([3, -1])
    assert torch.equal(c.d_pool[c.ids[1]], pool[c.ids[1]])
    assert ops.check_status() == 0


COMMIT = [
    # HK, HV, D, K, nodes, accepted, chain
    (2, 4, 128, 4, [1, 5, 8, 3], [0, 4, -1, 2], False),
    (1, 4, 64, 3, [3, 0, 16, 9], [2, -1, 15, 0], False),
    (3, 6, 128, 2, [64, 33], [63, 20], True),
    (1, 1, 64, 4, [64, 9, 8], [60, 8, 7], True),
    (2, 4, 128, 4, [40, 64, 17], [39, 63, 16], False),
]


@pytest.mark.parametrize("HK,HV,D,K,lens,accepted,chain", COMMIT)
def test_commit(ops, HK, HV, D, K, lens, accepted, chain):
    c = Gdn(HK, HV, D, lens, seed=sum(lens), K=K, chain=chain)
    c.commit(ops, accepted)
    c.check_pools(accepted)
    assert ops.check_status() == 0


def test_commit_accepts_strided_unaligned_rows(ops):
    c = Gdn(2, 4, 128, [6, 2], seed=21)
    for t in ("d_k", "d_v"):
        a = getattr(c, t)
        wide = torch.zeros(c.N, a.shape[1] * a.shape[2] + 1, dtype=torch.bfloat16, device=DEV)
        wide[:, 1:] = a.reshape(c.N, -1)
        setattr(c, t, wide[:, 1:].unflatten(1, a.shape[1:]))
    c.commit(ops, [5, 1])
    c.check_pools([5, 1])


@pytest.mark.parametrize("C,K,pdt", [(1024, 4, torch.float32), (96, 3, torch.bfloat16),
                                     (100, 2, torch.float32), (2056, 4, torch.float32)])
def test_conv_gate(ops, C, K, pdt):
    r = np.random.default_rng(C)
    lens, H = [5, 0, 64, 1, 2, 33], 6
    trees, n = R.make_trees(lens, C), sum(lens)
    pool, ids = rnd(r, 9, 2, C, K - 1), r.permutation(9)[:6]
    row, w = rnd(r, n + 4, C + 2 * H + 4), rnd(r, C, K, std=0.3)
    a_log, dt = rnd(r, H, std=0.5), rnd(r, H, std=0.5)
    dev, d_pool = bf(row), bf(pool)
    par = i32(np.concatenate(trees + [np.full(4, 99)]))
    args = (d_pool[:, 1], i64(ids), bf(w), i32(R.cu_of(lens)), par, 64, dev[:, C:C + H],
            dev[:, C + H:C + 2 * H], f32(a_log).to(pdt), f32(dt).to(pdt))
    y, g, beta = ops.conv_gate_tree(dev[:, :C], *args)
    ry, rg, rb = R.conv_gate(row[:n, :C], pool[ids, 1], w, trees, row[:n, C + H:C + 2 * H],
                             row[:n, C:C + H], a_log, dt)
    close(y[:n], ry, 2.0 ** -18, "y")
    close(beta[:n], rb, 2.0 ** -18, "beta")
    # g in fp32: exp, log and their product, a few units in 2^-23, relative to softplus's 1 + exp
    assert (np.abs(host(g[:n]) - rg) <= 2.0 ** -21 * (np.abs(rg) + np.exp(a_log))).all()
    assert np.array_equal(host(d_pool), pool), "the windows are only read"
    assert ops.check_status() == 0


@pytest.mark.parametrize("C", [1024, 100])
def test_conv_gate_chain_has_the_varlen_bits(ops, C):
    r = np.random.default_rng(7)
    lens, H, K = [9, 3, 64, 1], 4, 4
    n = sum(lens)
    dev, w = bf(rnd(r, n, C + 2 * H)), bf(rnd(r, C, K, std=0.3))
    pool, ids, cu = bf(rnd(r, 5, C, K - 1)), i64([3, 0, 4, 1]), i32(R.cu_of(lens))
    gate = (dev[:, C:C + H], dev[:, C + H:], f32(rnd(r, H)), f32(rnd(r, H)))
    par = i32(np.concatenate(R.make_trees(lens, 0, chain=True)))
    got = ops.conv_gate_tree(dev[:, :C], pool, ids, w, cu, par, 64, *gate)
    ref = ops.conv_gate_varlen(dev[:, :C], pool.clone(), ids, w, cu, *gate)
    for a, b in zip(got, ref):
        assert torch.equal(a, b)


def test_conv_gate_nan_stays_on_its_path(ops):
    c = Gdn(1, 2, 64, [12], seed=4, wide=3)
    args = (c.d_conv[:, 1], c.d_ids, bf(c.w), *c.tree, c.d_b, c.d_a, f32(c.a_log), f32(c.dt))
    ref = [t.clone() for t in ops.conv_gate_tree(c.d_x, *args)]
    c.d_x[3] = float("nan")
    got = ops.conv_gate_tree(c.d_x, *args)
    hit = torch.tensor([3 in R.ancestors(c.trees[0], i)[-4:] for i in range(12)], device=DEV)
    assert got[0][hit].isnan().all() and torch.equal(got[0][~hit], ref[0][~hit])


# ---------------------------------------------------------------------------
# the attention side
# ---------------------------------------------------------------------------


class Paged:
    """A paged cache with its tables; pages nobody owns, and the places behind the
    last node, hold NaN."""

    def __init__(self, HKV, D, block, ctx, lens, seed, spare=3):
        r = np.random.default_rng(seed)
        self.ctx, self.lens, self.block = ctx, lens, block
        pages = [-(-(c + n) // block) for c, n in zip(ctx, lens)]
        total = sum(pages) + spare
        order = r.permutation(total)
        self.table = np.full((len(ctx), max(pages + [0]) + 2), -1, np.int64)
        self.k, self.v = np.full((total, block, HKV, D), np.nan), np.full((total, block, HKV, D), np.nan)
        self.ks, self.vs, at = [], [], 0
        for s, m in enumerate(pages):
            own = order[at:at + m]
            self.table[s, :m] = own
            at += m
            n = ctx[s] + lens[s]
            k, v = rnd(r, n, HKV, D), rnd(r, n, HKV, D)
            self.ks.append(k)
            self.vs.append(v)
            p = np.arange(n)
            self.k[own[p // block], p % block], self.v[own[p // block], p % block] = k, v
        self.d_k, self.d_v, self.d_table, self.d_ctx = bf(self.k), bf(self.v), i32(self.table), i32(ctx)

    @property
    def most(self):
        return max(c + n for c, n in zip(self.ctx, self.lens))


def attn_close(got, ref, size):
    got = host(got)
    tol = U * np.abs(ref) + U * size + 1e-30
    bad = ~(np.abs(got - ref) <= tol)
    assert not bad.any(), f"{bad.sum()} of {bad.size}, worst {np.nanmax(np.abs(got - ref) / tol):.2f}, " \
        f"NaN {np.isnan(got).sum()}"


ATTN = [
    # HQ, HKV, D, block, contexts, nodes, chain
    (4, 1, 128, 256, [0, 1, 255, 256, 257], [1, 1, 1, 1, 1], True),
    (16, 4, 128, 256, [300, 0, 63, 64], [5, 8, 0, 3], False),
    (4, 4, 64, 16, [5, 100, 33], [2, 16, 7], False),
    (6, 2, 64, 48, [1000, 47, 0], [9, 1, 20], False),
    (8, 1, 128, 16, [513, 2], [64, 30], False),
    (8, 2, 256, 64, [200, 0, 31], [3, 4, 17], False),
    (2, 2, 256, 256, [700, 9], [64, 33], True),
    (16, 1, 64, 1, [70, 3], [2, 1], True),
    (4, 1, 128, 100, [1, 640], [32, 16], True),
]


@pytest.mark.parametrize("HQ,HKV,D,block,ctx,lens,chain", ATTN)
def test_attention(ops, HQ, HKV, D, block, ctx, lens, chain):
    seed = HQ + D + sum(ctx)
    c, trees = Paged(HKV, D, block, ctx, lens, seed), R.make_trees(lens, seed, chain)
    q = rnd(np.random.default_rng(seed), sum(lens), HQ, D)
    out = ops.attention_tree(bf(q), c.d_k, c.d_v, c.d_table, c.d_ctx, i32(R.cu_of(lens)),
                             i32(np.concatenate(trees)), max(lens), c.most)
    ref, size = R.attention(q, c.ks, c.vs, ctx, trees, D ** -0.5)
    attn_close(out, ref, size)
    assert ops.check_status() == 0


@pytest.mark.parametrize("D,nodes,HQ", [(128, 1, 4), (128, 7, 4), (64, 40, 4), (256, 2, 2)])
def test_attention_long_context_over_many_ctas(ops, D, nodes, HQ):
    """Few sequences over long contexts: every unit is cut and joined afterwards."""
    ctx, lens = [9000, 4097], [nodes, 1]
    c, trees = Paged(1, D, 64, ctx, lens, 11), R.make_trees(lens, 3)
    q = rnd(np.random.default_rng(1), sum(lens), HQ, D, std=2.0)
    out = ops.attention_tree(bf(q), c.d_k, c.d_v, c.d_table, c.d_ctx, i32(R.cu_of(lens)),
                             i32(np.concatenate(trees)), nodes, 9100, scale=0.3)
    ref, size = R.attention(q, c.ks, c.vs, ctx, trees, 0.3)
    attn_close(out, ref, size)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("D,nodes,ctx", [(128, 6, 100), (64, 50, 0), (256, 12, 3000)])
def test_attention_nan_stays_on_its_path(ops, D, nodes, ctx, bad):
    lens = [nodes, 2]
    c, trees = Paged(2, D, 64, [ctx, 5], lens, 2), R.make_trees(lens, 8, wide=3)
    q = rnd(np.random.default_rng(1), sum(lens), 4, D)
    ref, size = R.attention(q, c.ks, c.vs, [ctx, 5], trees, D ** -0.5)
    at = ctx + 2
    page = c.table[0, at // 64]
    c.d_k[page, at % 64] = bad
    c.d_v[page, at % 64] = bad
    got = host(ops.attention_tree(bf(q), c.d_k, c.d_v, c.d_table, c.d_ctx, i32(R.cu_of(lens)),
                                  i32(np.concatenate(trees)), nodes, c.most))
    hit = np.array([2 in R.ancestors(trees[0], i) for i in range(nodes)] + [False] * 2)
    assert not np.isfinite(got[hit]).any()
    tol = U * (np.abs(ref) + size)
    assert (np.abs(got - ref)[~hit] <= tol[~hit]).all()


def test_attention_large_scores(ops):
    """Scores far apart and of the type's size: the running maximum carries them."""
    c, trees = Paged(1, 64, 16, [500], [3], 4), R.make_trees([3], 0)
    q = rnd(np.random.default_rng(0), 3, 2, 64, std=300.0)
    out = ops.attention_tree(bf(q), c.d_k, c.d_v, c.d_table, c.d_ctx, i32([0, 3]), i32(trees[0]),
                             3, c.most, scale=1.0)
    ref, size = R.attention(q, c.ks, c.vs, [500], trees, 1.0)
    attn_close(out, ref, size)


@pytest.mark.parametrize("D,rot,offset", [(64, 64, False), (128, 32, True), (128, 128, False),
                                          (256, 64, True), (64, 48, True)])
def test_qk_norm_rope(ops, D, rot, offset):
    r = np.random.default_rng(D + rot)
    HQ, HKV, block, blocks, n = 6, 2, 48, 5, 37
    row = rnd(r, n, (HQ + 2 * HKV) * D)
    q, k, v = np.split(row.reshape(n, -1, D), [HQ, HQ + HKV], 1)
    qw, kw = rnd(r, D), rnd(r, D)
    ang = r.uniform(0, 6.3, (4000, rot // 2))
    cs = np.concatenate([np.cos(ang), np.sin(ang)], 1).astype(np.float32)
    pos, slot = r.integers(0, 4000, n), r.permutation(blocks * block)[:n]
    slot[5] = -1
    # a cache that is one layer of a larger buffer: wide block strides
    kv = bf(rnd(r, 2, blocks, 3, block, HKV, D))
    kc, vc = kv[0][:, 1], kv[1][:, 1]
    before = kv.clone()
    d = bf(row).view(n, -1, D)
    out = ops.qk_norm_rope_cache(d[:, :HQ], d[:, HQ:HQ + HKV], d[:, HQ + HKV:], bf(qw), bf(kw),
                                 f32(cs), i64(pos), kc, vc, i32(slot), eps=1e-5, unit_offset=offset)
    c, s = cs[pos, :rot // 2].astype(np.float64), cs[pos, rot // 2:].astype(np.float64)
    close(out, R.norm_rope(q, qw, c, s, 1e-5, float(offset)), 2.0 ** -18, "q")
    rk = R.norm_rope(k, kw, c, s, 1e-5, float(offset))
    keep = slot >= 0
    close(kc[slot[keep] // block, slot[keep] % block], rk[keep], 2.0 ** -18, "k")
    assert np.array_equal(host(vc[slot[keep] // block, slot[keep] % block]), v[keep])
    mask = torch.ones(blocks, block, dtype=torch.bool, device=DEV)
    mask[slot[keep] // block, slot[keep] % block] = False
    assert torch.equal(kc[mask], before[0][:, 1][mask]) and torch.equal(vc[mask], before[1][:, 1][mask])
    assert torch.equal(kv[:, :, ::2], before[:, :, ::2]), "the buffer's other layers"
    assert ops.check_status() == 0


def test_qk_norm_rope_many_rows(ops):
    """Enough rows for the form with more heads per thread; both kinds of heads in one group."""
    r = np.random.default_rng(3)
    n, HQ, HKV, D, rot = 5000, 9, 2, 64, 32
    d = bf(rnd(r, n, HQ + 2 * HKV, D))
    qw, kw = rnd(r, D), rnd(r, D)
    ang = r.uniform(0, 6.3, (50, rot // 2))
    cs = np.concatenate([np.cos(ang), np.sin(ang)], 1).astype(np.float32)
    pos, slot = r.integers(0, 50, n), r.permutation(320 * 16)[:n]
    slot[::7] = -1
    kc, vc = (torch.zeros(320, 16, HKV, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    out = ops.qk_norm_rope_cache(d[:, :HQ], d[:, HQ:HQ + HKV], d[:, HQ + HKV:], bf(qw), bf(kw),
                                 f32(cs), i64(pos), kc, vc, i32(slot))
    c, s = cs[pos, :rot // 2].astype(np.float64), cs[pos, rot // 2:].astype(np.float64)
    x = host(d)
    close(out, R.norm_rope(x[:, :HQ], qw, c, s, 1e-6, 0), 2.0 ** -18, "q")
    keep = slot >= 0
    rk = R.norm_rope(x[:, HQ:HQ + HKV], kw, c, s, 1e-6, 0)
    close(kc.view(-1, HKV, D)[slot[keep]], rk[keep], 2.0 ** -18, "k")
    ref_v = torch.zeros_like(vc).view(-1, HKV, D)
    ref_v[slot[keep]] = d[:, HQ + HKV:][torch.from_numpy(keep)]
    assert torch.equal(vc.view(-1, HKV, D), ref_v) and ops.check_status() == 0


def test_qk_norm_rope_unaligned_rows_and_one_row(ops):
    r = np.random.default_rng(0)
    for n in (1, 3):
        wide = bf(rnd(r, n, 5 * 64 + 7))
        q, k, v = (wide[:, 1:129].view(n, 2, 64), wide[:, 129:193].view(n, 1, 64),
                   wide[:, 193:257].view(n, 1, 64))
        cs = f32(np.concatenate([np.ones((8, 8)), np.zeros((8, 8))], 1))
        kc, vc = (torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        out = ops.qk_norm_rope_cache(q, k, v, bf(np.ones(64)), bf(np.ones(64)), cs,
                                     i64(np.arange(n)), kc, vc, i32(np.arange(n)))
        close(out, R.norm_rope(host(q), np.ones(64), np.ones((n, 8)), np.zeros((n, 8)), 1e-6, 0), 2.0 ** -18)
        assert torch.equal(vc.view(8, 1, 64)[:n], v)


@pytest.mark.parametrize("accept", [False, True])
@pytest.mark.parametrize("block,lens", [(256, [1, 5, 3]), (16, [64, 0, 17, 64, 2, 33, 1]),
                                        (1, [4, 4]), (48, [1] * 300)])
def test_slot_map(ops, block, lens, accept):
    r = np.random.default_rng(block)
    trees, n = R.make_trees(lens, block), sum(lens)
    ctx = r.integers(0, 700, len(lens))
    table = r.permutation(len(lens) * (800 // block + 1)).reshape(len(lens), -1)
    acc = np.array([r.integers(-1, m) if m else -1 for m in lens])
    par = i32(np.concatenate(trees + [np.full(3, 5)]))
    pos, slot = ops.tree_slot_map(i32(table), i32(ctx), i32(R.cu_of(lens)), par, 64, block, n + 3,
                                  accepted=i32(acc) if accept else None)
    rp, rs = R.slots(table, ctx, trees, block, acc if accept else None)
    assert np.array_equal(pos[:n].cpu().numpy(), rp) and np.array_equal(slot[:n].cpu().numpy(), rs)
    assert (pos[n:] == 0).all() and (slot[n:] == -1).all()
    assert pos.dtype == torch.int64 and slot.dtype == torch.int32 and ops.check_status() == 0
