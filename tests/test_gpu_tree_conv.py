"""The conv along trees in both of its forms (four channels to a thread where sizes, strides
and addresses allow whole words of four, else one), and its activation far from zero.

Tolerances: those of test_gpu_tree.py.
"""
import numpy as np
import pytest
import torch

import _tree_reference as R
from test_gpu_tree import DEV, bf, close, f32, host, i32, i64, ops, rnd  # noqa: F401

pytestmark = pytest.mark.gpu
LENS, H = [5, 0, 64, 1, 2, 33], 6


class Conv:
    """Rows of `width` elements that hold x from element `lead` on."""

    def __init__(self, C, K, lead, width, chain, lens=LENS, seed=0):
        r = np.random.default_rng(C + K + seed)
        self.n, self.C, self.K, self.lens = sum(lens), C, K, lens
        self.trees = R.make_trees(lens, C, chain)
        self.pool, self.ids = rnd(r, 9, C, K - 1), r.permutation(9)[:len(lens)]
        self.row, self.w = rnd(r, self.n, width), rnd(r, C, K, std=0.3)
        self.ab, self.a_log, self.dt = rnd(r, self.n, 2 * H), rnd(r, H, std=0.5), rnd(r, H, std=0.5)
        self.d_row, self.d_pool, self.d_w = bf(self.row), bf(self.pool), bf(self.w)
        self.x, self.d_x = self.row[:, lead:lead + C], self.d_row[:, lead:lead + C]
        ab = bf(self.ab)
        self.gate = (ab[:, H:], ab[:, :H], f32(self.a_log), f32(self.dt))
        self.cu = i32(R.cu_of(lens))

    def tree(self, ops):  # noqa: F811
        return ops.conv_gate_tree(self.d_x, self.d_pool, i64(self.ids), self.d_w, self.cu,
                                  i32(np.concatenate(self.trees)), 64, *self.gate)

    def varlen(self, ops):  # noqa: F811
        live = [i for i, n in enumerate(self.lens) if n]
        cu = i32(R.cu_of([self.lens[i] for i in live]))
        return ops.conv_gate_varlen(self.d_x, self.d_pool.clone(), i64(self.ids[live]), self.d_w, cu,
                                    *self.gate)


# channels, first element and width of a row: an odd count, counts of whole pairs only, rows of an odd
# width, rows that begin in the middle of a word; the last one is the form of four
FORMS = [(99, 0, 99), (130, 0, 130), (66, 0, 66), (1, 0, 1), (100, 0, 101), (100, 1, 104), (256, 2, 264),
         (300, 4, 304)]


@pytest.mark.parametrize("K", [2, 3, 4])
@pytest.mark.parametrize("C,lead,width", FORMS)
def test_conv_forms(ops, C, lead, width, K):  # noqa: F811
    c = Conv(C, K, lead, width, chain=False)
    y, g, beta = c.tree(ops)
    ry, rg, rb = R.conv_gate(c.x, c.pool[c.ids], c.w, c.trees, c.ab[:, :H], c.ab[:, H:], c.a_log, c.dt)
    close(y, ry, 2.0 ** -18, "y")
    close(beta, rb, 2.0 ** -18, "beta")
    assert (np.abs(host(g) - rg) <= 2.0 ** -21 * (np.abs(rg) + np.exp(c.a_log))).all()
    assert np.array_equal(host(c.d_pool), c.pool) and ops.check_status() == 0


@pytest.mark.parametrize("K", [2, 3, 4])
@pytest.mark.parametrize("C,lead,width", FORMS)
def test_chains_have_the_varlen_bits(ops, C, lead, width, K):  # noqa: F811
    c = Conv(C, K, lead, width, chain=True)
    for a, b in zip(c.tree(ops), c.varlen(ops)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("C", [256, 99])
def test_the_activation_far_from_zero(ops, C):  # noqa: F811
    """One tap of weight one, so that what enters the activation is x itself: every bf16 value,
    infinities and NaN among them, against the other conv's bits and, where finite, the definition."""
    bits = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    n = -(-bits.numel() // C)
    lens = [64] * (n // 64) + [n % 64]
    x = torch.zeros(n * C, dtype=torch.bfloat16)
    x[:bits.numel()] = bits
    x = x.view(n, C).to(DEV)
    w = torch.zeros(C, 2, dtype=torch.bfloat16, device=DEV)
    w[:, 1] = 1
    pool = torch.zeros(len(lens), C, 1, dtype=torch.bfloat16, device=DEV)
    ids = torch.arange(len(lens), device=DEV)
    gate = (x[:, :1], x[:, :1], f32([0.0]), f32([0.0]))
    roots = torch.full((n,), -1, dtype=torch.int32, device=DEV)
    cu = i32(R.cu_of(lens))
    y = ops.conv_gate_tree(x, pool, ids, w, cu, roots, 64, *gate)[0]
    # the other conv sees the row before through a weight of zero: rows of their own
    ones = i32(np.arange(n + 1))
    many = torch.zeros(n, C, 1, dtype=torch.bfloat16, device=DEV)
    want = ops.conv_gate_varlen(x, many, torch.arange(n, device=DEV), w, ones, *gate)[0]
    assert torch.equal(y.isnan(), want.isnan())
    assert torch.equal(y.nan_to_num(7.0).view(torch.int16), want.nan_to_num(7.0).view(torch.int16))
    v = host(x)
    fine = np.isfinite(v)
    v = np.where(fine, v, 0.0)
    ref = np.where(v >= 0, v / (1 + np.exp(-np.maximum(v, 0))), v * np.exp(np.minimum(v, 0)) / (1 + np.exp(np.minimum(v, 0))))
    # half a step, 2^-18 of the arithmetic, and below 2^-126 / 2^-125 (flushed products) nothing
    tol = (2.0 ** -8 + 2.0 ** -18) * np.abs(ref) + 2.0 ** -117
    assert (np.abs(host(y) - ref)[fine] <= tol[fine]).all()


@pytest.mark.parametrize("K", [2, 4])
def test_chains_have_the_varlen_bits_far_from_zero(ops, K):  # noqa: F811
    """fp32 sums in front of the activation from 2^-20 to 1000 in size, of both signs."""
    r = np.random.default_rng(K)
    C, lens = 1024, [64] * 30
    c = Conv(C, K, 0, C, chain=True, lens=lens[:6])
    n = sum(lens)
    x = torch.from_numpy((rnd(r, n, C) * 2.0 ** r.uniform(-20, 8, (n, 1))).astype(np.float32)).to(torch.bfloat16).to(DEV)
    w, pool = bf(rnd(r, C, K)), bf(rnd(r, len(lens), C, K - 1))
    ids, cu = torch.arange(len(lens), device=DEV), i32(R.cu_of(lens))
    gate = (x[:, :H], x[:, :H], c.gate[2], c.gate[3])
    par = i32(np.concatenate(R.make_trees(lens, 0, chain=True)))
    got = ops.conv_gate_tree(x, pool, ids, w, cu, par, 64, *gate)
    want = ops.conv_gate_varlen(x, pool.clone(), ids, w, cu, *gate)
    assert got[0].isfinite().all() and got[0].abs().max() > 500 and (got[0] == 0).any()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
