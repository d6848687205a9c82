"""64-bit restatements of the tree operators, one sequence and one node after
the other, for the tests of the kernels (numpy on the CPU)."""
import numpy as np

L2_EPS = 1e-6


def ancestors(parents, i):
    """Node i and its ancestors, the root first."""
    path = []
    while i >= 0:
        path.insert(0, i)
        i = parents[i]
    return path


def make_trees(lens, seed, chain=False, wide=4):
    """Parents of every row (relative to its sequence), one array per sequence."""
    r = np.random.default_rng(seed)
    out = []
    for n in lens:
        p = np.full(n, -1, np.int64)
        for i in range(1, n):
            p[i] = i - 1 if chain else r.integers(max(-1, i - wide), i)
        out.append(p)
    return out


def cu_of(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)


def silu(x):
    return x / (1.0 + np.exp(-x))


def conv_gate(x, windows, w, trees, a, b, a_log, dt_bias):
    """windows: [n_seqs, C, K-1] of the sequences' slots."""
    y, at = np.zeros(x.shape), 0
    for r, par in enumerate(trees):
        for i in range(len(par)):
            rows = [x[at + j] for j in ancestors(par, i)]
            full = np.concatenate([windows[r], np.stack(rows, 1)], 1)[:, -w.shape[1]:]
            y[at + i] = (full * w).sum(1)
        at += len(par)
    z = a + dt_bias
    g = -np.exp(a_log) * np.where(z > 20, z, np.log1p(np.exp(np.minimum(z, 20))))
    return silu(y), g, 1 / (1 + np.exp(-b))


def l2norm(x):
    return x / np.sqrt((x * x).sum(-1, keepdims=True) + L2_EPS)


def step(S, k, v, g, beta):
    """One token of one head set: S [HV, DK, DV], k / v [HV, D], g / beta [HV]."""
    S = S * np.exp(g)[:, None, None]
    d = beta[:, None] * (v - np.einsum("hkv,hk->hv", S, k))
    return S + k[:, :, None] * d[:, None, :]


def delta(q, k, v, g, beta, states, trees, z=None, w=None, eps=1e-6):
    """states [n_seqs, HV, DK, DV]; q / k [N, HK, DK]; returns [N, HV, DV]."""
    HV, D = v.shape[1], v.shape[2]
    rep = HV // q.shape[1]
    qn, kn = l2norm(q).repeat(rep, 1) * q.shape[2] ** -0.5, l2norm(k).repeat(rep, 1)
    out, at = np.zeros(v.shape), 0
    for r, par in enumerate(trees):
        after = []
        for i, p in enumerate(par):
            S = step(states[r] if p < 0 else after[p], kn[at + i], v[at + i], g[at + i],
                     beta[at + i])
            after.append(S)
            out[at + i] = np.einsum("hkv,hk->hv", S, qn[at + i])
        at += len(par)
    if z is not None:
        out = out / np.sqrt((out * out).mean(-1, keepdims=True) + eps) * w * silu(z)
    return out


def commit(x, k, v, g, beta, windows, states, trees, accepted):
    """(windows, states) of every sequence after its accepted path."""
    rep = v.shape[1] // k.shape[1]
    kn = l2norm(k).repeat(rep, 1)
    windows, states, at = windows.copy(), states.copy(), 0
    for r, par in enumerate(trees):
        path = [at + i for i in ancestors(par, accepted[r])]
        for n in path:
            states[r] = step(states[r], kn[n], v[n], g[n], beta[n])
        if path:
            windows[r] = np.concatenate([windows[r], x[path].T], 1)[:, -windows.shape[2]:]
        at += len(par)
    return windows, states


def norm_rope(x, w, cos, sin, eps, offset):
    """x [N, H, D]; cos / sin [N, R / 2]."""
    x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (w + offset)
    h = cos.shape[1]
    a, b = x[..., :h], x[..., h:2 * h]
    c, s = cos[:, None], sin[:, None]
    return np.concatenate([a * c - b * s, b * c + a * s, x[..., 2 * h:]], -1)


def attention(q, ks, vs, ctx, trees, scale):
    """ks / vs: per sequence [context + nodes, HKV, D].  Returns the outputs and the
    same weights over |v| (the size of what was summed)."""
    out, size, at = np.zeros(q.shape), np.zeros(q.shape), 0
    for r, par in enumerate(trees):
        for i in range(len(par)):
            cols = list(range(ctx[r])) + [ctx[r] + j for j in ancestors(par, i)]
            for h in range(q.shape[1]):
                kv = h // (q.shape[1] // ks[r].shape[1])
                s = ks[r][cols, kv] @ q[at + i, h] * scale
                p = np.exp(s - s.max())
                p /= p.sum()
                out[at + i, h] = p @ vs[r][cols, kv]
                size[at + i, h] = p @ np.abs(vs[r][cols, kv])
        at += len(par)
    return out, size


def slots(table, ctx, trees, block, accepted=None):
    pos, slot = [], []
    for r, par in enumerate(trees):
        path = ancestors(par, accepted[r]) if accepted is not None else None
        for i in range(len(par)):
            depth = len(ancestors(par, i)) - 1
            pos.append(ctx[r] + depth)
            at = ctx[r] + (i if path is None else depth)
            ok = path is None or i in path
            slot.append(table[r][at // block] * block + at % block if ok else -1)
    return np.array(pos, np.int64), np.array(slot, np.int32)
