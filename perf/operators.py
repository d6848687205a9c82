"""The operators that check drafted tokens in the hybrid decoder, and their measured cases.

A server that drafts tokens has, for each sequence, a small tree of them: node 0 is the last token that it
holds for sure, every other node hangs under an earlier one.  One pass computes all nodes, the sampler says
which path stands, and that path is taken over.  The gated-delta-rule layers keep a recurrent state and a
conv window for each sequence, which a rejected token must not touch; the attention layers keep a paged
cache.  Six operators do this work:

* ``conv_gate``  causal conv along each node's ancestors, back into the sequence's stored window, with the
                 decay gate and write strength; the stored window stays as it is
* ``delta``      the gated delta rule along each node's ancestors from the stored state, gated norm included;
                 the stored state stays as it is
* ``commit``     takes the accepted path into the conv window and the recurrent state
* ``qk_rope``    RMS norm of every query and key head, the position rotation, and keys and values into the
                 paged cache
* ``attention``  every node against its sequence's paged cache and its own ancestors
* ``slots``      positions and cache slots of the nodes, before the pass and after acceptance

A case is a dict of plain values.  ``nodes`` bounds a sequence's tree; the sequences' own sizes go from
``nodes_lo`` to it.  ``tree`` false makes every tree a chain.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
EPS = 1e-6


def listed():
    gdn = {"hk": 16, "hv": 32, "d": 128, "taps": 4}          # the layer's full head shapes
    att = {"hq": 16, "hkv": 4, "d": 128, "block": 256}       # the hybrid decoder's attention layers
    return [
        # one user, a short chain: the call is as long as its launch
        {"name": "conv gate, 1 x 5 chain", "op": "conv_gate", "bs": 1, "nodes_lo": 5, "nodes": 5, "tree": False, "layers": 2, **gdn},
        # a full server with wide trees of uneven size
        {"name": "conv gate, 128 x 17..64", "op": "conv_gate", "bs": 128, "nodes_lo": 17, "nodes": 64, "tree": True, "layers": 1, **gdn},
        # a handful of users
        {"name": "delta, 4 x 5 chain", "op": "delta", "bs": 4, "nodes_lo": 5, "nodes": 5, "tree": False, "layers": 2, **gdn},
        # the full decode batch, a tree of up to eight nodes each: the states are the traffic
        {"name": "delta, 256 x 3..8", "op": "delta", "bs": 256, "nodes_lo": 3, "nodes": 8, "tree": True, "layers": 1, **gdn},
        # one shard of a head-sharded layer with few users
        {"name": "commit, 8 x 7, shard", "op": "commit", "bs": 8, "nodes_lo": 7, "nodes": 7, "tree": True, "layers": 2, "hk": 2, "hv": 4, "d": 128, "taps": 4},
        # the full decode batch
        {"name": "commit, 256 x 3..8", "op": "commit", "bs": 256, "nodes_lo": 3, "nodes": 8, "tree": True, "layers": 1, **gdn},
        # a plain decode step of 128 sequences, a quarter of each head rotated
        {"name": "qk rope, 128 x 1", "op": "qk_rope", "bs": 128, "nodes_lo": 1, "nodes": 1, "tree": False, "ctx_lo": 256, "ctx": 4352, "rot": 32, **att},
        # wide trees: some eight thousand rows, whole heads rotated
        {"name": "qk rope, 192 x 24..63", "op": "qk_rope", "bs": 192, "nodes_lo": 24, "nodes": 63, "tree": True, "ctx_lo": 1, "ctx": 1000, "rot": 128, **att},
        # the hybrid decoder's decode step: one token for each of 128 sequences, contexts of 256 to 4352
        {"name": "attention, 128 x 1", "op": "attention", "bs": 128, "nodes_lo": 1, "nodes": 1, "tree": False, "ctx_lo": 256, "ctx": 4352, **att},
        # trees over long prompts: up to 32 nodes against 4 to 8 thousand cached tokens
        {"name": "attention, 32 x 16..32", "op": "attention", "bs": 32, "nodes_lo": 16, "nodes": 32, "tree": True, "ctx_lo": 4096, "ctx": 8192, **att},
        # slots of a chain before its pass
        {"name": "slots, 5 x 5 chain", "op": "slots", "bs": 5, "nodes_lo": 5, "nodes": 5, "tree": False, "ctx_lo": 100, "ctx": 3000, "block": 256, "accept": False},
        # slots of a full server's trees after acceptance
        {"name": "slots, 256 x 9..64", "op": "slots", "bs": 256, "nodes_lo": 9, "nodes": 64, "tree": True, "ctx_lo": 1, "ctx": 8192, "block": 16, "accept": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["conv_gate", "delta", "commit", "qk_rope", "attention", "slots"])
    nodes = _log(rng, 1, 64)
    case = {"op": op, "nodes_lo": rng.randint(1, nodes), "nodes": nodes, "tree": rng.random() < 0.7}
    if op in ("conv_gate", "delta", "commit"):
        case["hk"], case["hv"] = rng.choice([(16, 32), (8, 16), (2, 4), (4, 8), (4, 4), (1, 4), (3, 6)])
        case["d"] = rng.choice([128, 128, 64])
        case["taps"] = rng.choice([4, 4, 3, 2])
        case["layers"] = rng.choice([1, 2])
        case["bs"] = _log(rng, 1, max(1, min(256 // case["layers"], (2048 if op != "conv_gate" else 5120) // nodes)))
        return case
    case["block"] = rng.choice([256, 256, 64, 16, 48])
    if op == "slots":
        case["bs"] = _log(rng, 1, 256)
        case["ctx_lo"], case["ctx"], case["accept"] = 0, _log(rng, 1, 8192), rng.random() < 0.5
        return case
    case["hq"], case["hkv"] = rng.choice([(16, 4), (16, 4), (8, 1), (4, 2), (4, 4), (6, 2)])
    case["d"] = rng.choice([128, 128, 64, 256])
    if op == "qk_rope":
        case["rot"] = rng.choice([case["d"], case["d"] // 2, case["d"] // 4])
        case["ctx_lo"], case["ctx"] = 0, _log(rng, 1, 2000)
        case["bs"] = _log(rng, 1, max(1, min(192, (1 << 24) // (nodes * case["hq"] * case["d"]))))
        return case
    # at most the listed trees' products and cached tokens
    per_token = nodes * case["hq"] * case["d"]
    case["ctx"] = _log(rng, 1, min(131072, (9 << 30) // per_token - nodes))
    case["ctx_lo"] = rng.randint(0, case["ctx"])
    kv = case["ctx"] + nodes
    case["bs"] = _log(rng, 1, max(1, min(128, (3 << 25) // (kv * case["hkv"] * case["d"]), (9 << 30) // (kv * per_token))))
    return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _spread(n, lo, hi):
    """n whole numbers from lo to hi, the same ones for every seed."""
    i = np.arange(1, n + 1, dtype=np.uint64)
    return (lo + ((i * np.uint64(2654435761) & np.uint64(0xFFFFFFFF)) * np.uint64(hi - lo + 1) >> np.uint64(32)).astype(np.int64)).astype(np.int64)


def _sizes(case):
    lens = _spread(case["bs"], case["nodes_lo"], case["nodes"])
    ctx = _spread(case["bs"] + 3, case["ctx_lo"], case["ctx"])[3:] if "ctx" in case else None
    return lens, ctx


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rng = np.random.default_rng(seed)
    lens, ctx = _sizes(case)
    bs, op = case["bs"], case["op"]
    n = int(lens.sum())

    def nrm(*shape, std=1.0, dtype=torch.bfloat16):
        return torch.randn(*shape, generator=gen, device=DEV, dtype=dtype).mul_(std)

    def dev(a, dtype):
        return torch.from_numpy(np.ascontiguousarray(a)).to(DEV, dtype)

    parents, accepted = [], []
    for m in lens:
        i = np.arange(m)
        parents.append(np.where(i > 0, i - 1 - (rng.integers(0, np.maximum(np.minimum(i, 4), 1)) if case["tree"] else 0), -1))
        accepted.append(rng.integers(0, m))
    s = {"case": case, "cu": dev(np.concatenate([[0], np.cumsum(lens)]), torch.int32), "parents": dev(np.concatenate(parents), torch.int32),
         "accepted": dev(np.array(accepted), torch.int32), "n": n}
    if op in ("conv_gate", "delta", "commit"):
        hk, hv, d, taps = case["hk"], case["hv"], case["d"], case["taps"]
        c = (2 * hk + hv) * d
        slots = bs + 3
        s["ids"] = dev(rng.permutation(slots)[:bs], torch.int64)
        # one projection output holds all of a row: [q | k | v], z, b, a, and padding to a multiple of eight
        row = nrm(n, (c + hv * d + 2 * hv + 7) // 8 * 8)
        s["x"], s["z"] = row[:, :c], row[:, c:c + hv * d].view(n, hv, d)
        s["b"], s["a"] = row[:, c + hv * d:c + hv * d + hv], row[:, c + hv * d + hv:c + hv * d + 2 * hv]
        s["conv_pool"] = nrm(slots, case["layers"], c, taps - 1)
        s["conv"] = s["conv_pool"][:, case["layers"] - 1]
        s["w"] = (torch.rand(c, taps, generator=gen, device=DEV) - 0.5).to(torch.bfloat16)
        s["a_log"] = -torch.rand(hv, generator=gen, device=DEV)
        s["dt_bias"] = torch.zeros(hv, device=DEV)
        if op != "conv_gate":
            y = torch.nn.functional.silu(nrm(n, c, std=0.6, dtype=torch.float32)).to(torch.bfloat16)
            s["q"], s["k"], s["v"] = y[:, :hk * d].view(n, hk, d), y[:, hk * d:2 * hk * d].view(n, hk, d), y[:, 2 * hk * d:].view(n, hv, d)
            s["g"] = -torch.nn.functional.softplus(nrm(n, hv, dtype=torch.float32)) * s["a_log"].exp()
            s["beta"] = torch.sigmoid(nrm(n, hv, dtype=torch.float32)).to(torch.bfloat16)
            s["s_pool"] = nrm(slots, case["layers"], hv, d, d, std=0.02, dtype=torch.float32)
            s["state"] = s["s_pool"][:, case["layers"] - 1]
            s["norm_w"] = (1 + nrm(d, std=0.1, dtype=torch.float32)).to(torch.bfloat16)
        return s
    block = case["block"]
    pages = -(-(ctx + lens) // block)
    total = int(pages.sum()) + 2
    order, table, at = rng.permutation(total), np.full((bs, int(pages.max()) + 1), -1), 0
    for r, m in enumerate(pages):
        table[r, :m] = order[at:at + m]
        at += m
    s["table"], s["ctx"] = dev(table, torch.int32), dev(ctx, torch.int32)
    if op == "slots":
        return s
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    cache = nrm(2, total, block, hkv, d)
    s["k_cache"], s["v_cache"] = cache[0], cache[1]
    s["most"] = int((ctx + lens).max())
    if op == "attention":
        s["q"] = nrm(n, hq, d)
        return s
    row = nrm(n, (hq + 2 * hkv) * d)
    s["q"], s["k"], s["v"] = row[:, :hq * d].view(n, hq, d), row[:, hq * d:(hq + hkv) * d].view(n, hkv, d), row[:, (hq + hkv) * d:].view(n, hkv, d)
    s["q_w"], s["k_w"] = nrm(d, std=0.1), nrm(d, std=0.1)         # weights around zero: the norm scales by 1 + w
    freq = 1e6 ** (-torch.arange(0, case["rot"], 2, device=DEV, dtype=torch.float64) / case["rot"])
    angle = torch.arange(s["most"], device=DEV, dtype=torch.float64)[:, None] * freq
    s["cos_sin"] = torch.cat([angle.cos(), angle.sin()], 1).float()
    depth, pos, slot, at = [], [], [], 0
    for r, m in enumerate(lens):
        dep = np.zeros(m, np.int64)
        for i in range(1, m):
            dep[i] = dep[parents[r][i]] + 1
        pos.append(ctx[r] + dep)
        p = ctx[r] + np.arange(m)
        slot.append(table[r, p // block] * block + p % block)
    s["pos"], s["slot"] = dev(np.concatenate(pos), torch.int64), dev(np.concatenate(slot), torch.int32)
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------


def _rows(s):
    """Each row's sequence and its number there."""
    row = torch.arange(s["n"], device=DEV)
    seq = torch.searchsorted(s["cu"], row, right=True, out_int32=True).long() - 1
    return row, seq, row - s["cu"].long()[seq]


def _dense(s):
    """(index [bs, T] of the padded rows, live [bs, T], ancestors-or-self [bs, T, T])."""
    cu, t = s["cu"].long(), s["case"]["nodes"]
    i = torch.arange(t, device=DEV)
    live = i < (cu[1:] - cu[:-1])[:, None]
    index = torch.where(live, cu[:-1, None] + i, 0)
    up = torch.where(live, s["parents"].long()[index], -1)[:, :, None] == i
    closure = torch.linalg.matrix_power(up.float() + torch.eye(t, device=DEV), t) > 0
    return index, live, closure & live[:, :, None]


def _plain_conv_gate(s):
    taps, x, cu = s["case"]["taps"], s["x"].float(), s["cu"].long()
    row, seq, _ = _rows(s)
    start = cu[seq]
    up = torch.where(s["parents"] < 0, -1, start + s["parents"])
    up = torch.cat([up, up.new_tensor([-1])])                    # the last entry: above the root
    window, w = s["conv"][s["ids"]][seq].float(), s["w"].float()
    at, found, acc = row, torch.zeros_like(row), 0
    for i in range(taps):
        held = window.gather(2, (taps - 2 - (i - found)).clamp(0, taps - 2)[:, None, None].expand(-1, x.shape[1], 1))[:, :, 0]
        acc = acc + torch.where((at >= 0)[:, None], x[at], held) * w[:, taps - 1 - i]
        found = found + (at >= 0)
        at = up[at]
    z = s["a"].float() + s["dt_bias"]
    g = -s["a_log"].exp() * torch.where(z > 20, z, torch.log1p(z.exp()))
    return (acc * torch.sigmoid(acc)).to(torch.bfloat16), g, torch.sigmoid(s["b"].float()).to(torch.bfloat16)


def _solve(s):
    """What the delta rule makes of every node: (decay from the stored state [bs, h, T], decay between nodes
    and normed products [bs, h, T, T], the nodes' updates [bs, h, T, d], the stored states, ...)."""
    c = s["case"]
    index, live, anc = _dense(s)
    rep = c["hv"] // c["hk"]
    heads = lambda t: t[index].float().transpose(1, 2)           # [bs, heads, T, d]
    q, k, v = heads(s["q"]).repeat_interleave(rep, 1), heads(s["k"]).repeat_interleave(rep, 1), heads(s["v"])
    q = q * torch.rsqrt((q * q).sum(-1, keepdim=True) + EPS) * c["d"] ** -0.5
    k = k * torch.rsqrt((k * k).sum(-1, keepdim=True) + EPS)
    beta = s["beta"][index].float().transpose(1, 2)[..., None]
    # the decays' logarithms are summed and subtracted in 64 bits
    sums = (anc.double()[:, None] * s["g"][index].double().transpose(1, 2)[:, :, None]).sum(-1)
    anc = anc[:, None]
    between = torch.where(anc, (sums[..., None] - sums[..., None, :]).clamp(max=0.0).exp().float(), 0)
    first = sums.exp().float()[..., None]
    state = s["state"][s["ids"]]
    own_row = torch.eye(c["nodes"], device=DEV, dtype=torch.bool)
    low = torch.where(own_row, 0, -beta * between * (k @ k.transpose(-1, -2)))
    # (1 - low)^-1 as a product: low's power of the number of nodes is zero
    inv, power = torch.eye(c["nodes"], device=DEV) + low, low
    for _ in range(max(0, (c["nodes"] - 1).bit_length() - 1)):
        power = power @ power
        inv = inv + inv @ power
    update = inv @ (beta * (v - first * (k @ state)))
    return index, live, anc, q, k, between, first, state, update


def _plain_delta(s):
    index, live, anc, q, k, between, first, state, update = _solve(s)
    o = first * (q @ state) + (between * (q @ k.transpose(-1, -2))) @ update
    o = o.transpose(1, 2)[live]                                  # [rows, heads, d]
    z = s["z"].float()
    o = o * torch.rsqrt((o * o).mean(-1, keepdim=True) + EPS) * s["norm_w"].float() * z * torch.sigmoid(z)
    return o.to(torch.bfloat16)


def _plain_commit(s):
    c, taps = s["case"], s["case"]["taps"]
    index, live, anc, q, k, between, first, state, update = _solve(s)
    last = s["accepted"].long()[:, None, None, None]
    decay = between.gather(2, last.expand(-1, c["hv"], 1, c["nodes"]))[:, :, 0, :, None]
    s["state"][s["ids"]] = first.gather(2, last.expand(-1, c["hv"], 1, 1)) * state + (k * decay).transpose(-1, -2) @ update
    # the window keeps the last taps - 1 of (window, path)
    path = anc[:, 0].gather(1, s["accepted"].long()[:, None, None].expand(-1, 1, c["nodes"]))[:, 0]
    window = s["conv"][s["ids"]]
    every = torch.cat([window, s["x"][index].transpose(1, 2)], 2)
    held = torch.cat([path.new_ones(c["bs"], taps - 1), path], 1)
    rank = held.flip(1).cumsum(1).flip(1)                        # 1 for the last one held
    slot = torch.where(held & (rank < taps), taps - 1 - rank, taps - 1)
    new = every.new_zeros(every.shape[0], every.shape[1], taps)
    new.scatter_(2, slot[:, None].expand_as(every), every)
    s["conv"][s["ids"]] = new[:, :, :taps - 1]
    return s["s_pool"], s["conv_pool"]


def _plain_qk_rope(s):
    rot = s["case"]["rot"]
    cos, sin = s["cos_sin"][s["pos"]][:, None].chunk(2, -1)

    def one(x, w):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * (1 + w.float())
        a, b, rest = x[..., :rot // 2], x[..., rot // 2:rot], x[..., rot:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1).to(torch.bfloat16)

    block, slot = s["case"]["block"], s["slot"].long()
    s["k_cache"][slot // block, slot % block] = one(s["k"], s["k_w"])
    s["v_cache"][slot // block, slot % block] = s["v"]
    return one(s["q"], s["q_w"]), s["k_cache"], s["v_cache"]


def _plain_attention(s):
    c = s["case"]
    index, live, anc = _dense(s)
    bs, t, hkv, d = c["bs"], c["nodes"], c["hkv"], c["d"]
    at = torch.arange(s["most"], device=DEV)
    page = s["table"].long()[:, at // c["block"]].clamp(min=0)
    k, v = s["k_cache"][page, at % c["block"]], s["v_cache"][page, at % c["block"]]
    q = s["q"][index].float().view(bs, t, hkv, -1, d).permute(0, 2, 3, 1, 4).reshape(bs, hkv, -1, d)
    node = at - s["ctx"].long()[:, None]                         # the cached position's node, where it is one
    seen = anc.gather(2, node.clamp(0, t - 1)[:, None].expand(-1, t, -1)) & (node < t)[:, None] | (node < 0)[:, None]
    score = q @ k.permute(0, 2, 3, 1).float() * d ** -0.5
    score = torch.where(seen[:, None, None], score.view(bs, hkv, -1, t, s["most"]), -math.inf).view_as(score)
    p = (score - score.amax(-1, keepdim=True)).exp()
    o = (p @ v.permute(0, 2, 1, 3).float()) / p.sum(-1, keepdim=True)
    return o.view(bs, hkv, -1, t, d).permute(0, 3, 1, 2, 4).reshape(bs, t, -1, d)[live].to(torch.bfloat16)


def _plain_slots(s):
    c = s["case"]
    row, seq, node = _rows(s)
    index, live, anc = _dense(s)
    depth = (anc.sum(-1) - 1)[live]
    pos = s["ctx"].long()[seq] + depth
    if c["accept"]:
        kept = anc.gather(1, s["accepted"].long()[:, None, None].expand(-1, 1, c["nodes"]))[:, 0][live]
        at = pos
    else:
        kept, at = torch.ones_like(row, dtype=torch.bool), s["ctx"].long()[seq] + node
    slot = s["table"].long()[seq, at // c["block"]] * c["block"] + at % c["block"]
    return pos, torch.where(kept, slot, -1).to(torch.int32)


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------


def _ops():
    import __graft_entry__
    return __graft_entry__.load_package().ops


def _own(s):
    ops, c, op = _ops(), s["case"], s["case"]["op"]
    tree = (s["cu"], s["parents"], c["nodes"])
    if op == "conv_gate":
        return ops.conv_gate_tree(s["x"], s["conv"], s["ids"], s["w"], *tree, s["b"], s["a"], s["a_log"], s["dt_bias"])
    if op == "delta":
        return ops.gated_delta_rule_tree(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"], s["ids"], *tree, z=s["z"], norm_weight=s["norm_w"], eps=EPS)
    if op == "commit":
        ops.commit_tree(s["x"], s["k"], s["v"], s["g"], s["beta"], s["conv"], s["state"], s["ids"], *tree, s["accepted"])
        return s["s_pool"], s["conv_pool"]
    if op == "qk_rope":
        q = ops.qk_norm_rope_cache(s["q"], s["k"], s["v"], s["q_w"], s["k_w"], s["cos_sin"], s["pos"], s["k_cache"], s["v_cache"], s["slot"], eps=EPS, unit_offset=True)
        return q, s["k_cache"], s["v_cache"]
    if op == "attention":
        return ops.attention_tree(s["q"], s["k_cache"], s["v_cache"], s["table"], s["ctx"], *tree, s["most"])
    return ops.tree_slot_map(s["table"], s["ctx"], *tree, c["block"], s["n"], accepted=s["accepted"] if c["accept"] else None)


_PLAIN = {"conv_gate": _plain_conv_gate, "delta": _plain_delta, "commit": _plain_commit, "qk_rope": _plain_qk_rope,
          "attention": _plain_attention, "slots": _plain_slots}


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["case"]["op"]](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------


def work(case):
    lens, ctx = _sizes(case)
    bs, n, op = case["bs"], int(lens.sum()), case["op"]
    tree = 4 * n + 4 * (bs + 1)
    if op in ("conv_gate", "delta", "commit"):
        hk, hv, d, taps = case["hk"], case["hv"], case["d"], case["taps"]
        c = (2 * hk + hv) * d
        if op == "conv_gate":
            return {"bytes": n * c * 4 + bs * c * (taps - 1) * 2 + c * taps * 2 + n * hv * (4 + 6) + tree, "flops": n * c * (2 * taps + 4)}
        state = bs * hv * d * d * 4
        if op == "delta":
            # every node's query and key through the stored state
            return {"bytes": state + n * (c + 2 * hv * d) * 2 + n * hv * 6 + tree, "flops": 4 * n * hv * d * d}
        # about half of a tree's nodes are on the accepted path at most: counted as one node for each sequence
        return {"bytes": 2 * state + bs * ((hk + hv) * d * 2 + hv * 6) + bs * c * (taps - 1) * 4 + tree, "flops": 6 * bs * hv * d * d}
    if op == "slots":
        return {"bytes": tree + 8 * bs + n * (4 + 8 + 4), "flops": 0}
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if op == "qk_rope":
        return {"bytes": n * (hq + 2 * hkv) * d * 4 + n * (case["rot"] * 4 + 12), "flops": n * (hq + hkv) * d * 8}
    seen = int((ctx * lens).sum()) + n
    pages = int((-(-(ctx + lens) // case["block"])).sum())
    return {"bytes": int((ctx + lens).sum()) * hkv * d * 4 + 2 * n * hq * d * 2 + 4 * pages + tree, "flops": 4 * seen * hq * d}


# ---------------------------------------------------------------------------
# the definitions in 64 bits, one sequence and one node after the other
# ---------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    lens, _ = _sizes(case)
    op, start = case["op"], np.concatenate([[0], np.cumsum(lens)])
    parents = s["parents"].tolist()
    if op in ("conv_gate", "delta", "commit"):
        return _exact_gdn(s, case, lens, start, parents)
    block = case["block"]
    table, ctx, accepted = s["table"].tolist(), s["ctx"].tolist(), s["accepted"].tolist()
    if op == "slots":
        pos, slot = [], []
        for r, m in enumerate(lens):
            depth = []
            for i in range(m):
                p = parents[start[r] + i]
                depth.append(0 if p < 0 else depth[p] + 1)
            path, i = set(), accepted[r]
            while i >= 0:
                path.add(i)
                i = parents[start[r] + i]
            for i in range(m):
                pos.append(ctx[r] + depth[i])
                at = ctx[r] + (depth[i] if case["accept"] else i)
                slot.append(table[r][at // block] * block + at % block if i in path or not case["accept"] else -1)
        return torch.tensor(pos, device=DEV), torch.tensor(slot, dtype=torch.int32, device=DEV)
    if op == "qk_rope":
        rot = case["rot"]
        half = s["cos_sin"].double()[s["pos"]].unsqueeze(1)
        turn = torch.complex(half[..., :rot // 2].contiguous(), half[..., rot // 2:].contiguous())

        def one(x, w):
            x = x.double()
            x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * (w.double() + 1)
            r = torch.complex(x[..., :rot // 2].contiguous(), x[..., rot // 2:rot].contiguous()) * turn
            return torch.cat([r.real, r.imag, x[..., rot:]], -1)

        k, v, slot = s["k_cache"].double(), s["v_cache"].double(), s["slot"].long()
        k.view(-1, *k.shape[2:])[slot] = one(s["k"], s["k_w"])
        v.view(-1, *v.shape[2:])[slot] = s["v"].double()
        return one(s["q"], s["q_w"]), k, v
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    rep = case["hq"] // case["hkv"]
    for r, m in enumerate(lens):
        at = torch.arange(ctx[r] + int(m), device=DEV)
        where = (s["table"][r].long()[at // block], at % block)
        k, v = s["k_cache"][where].double(), s["v_cache"][where].double()
        seen = torch.zeros(int(m), ctx[r] + int(m), dtype=torch.bool)
        seen[:, :ctx[r]] = True
        for i in range(m):
            j = i
            while j >= 0:
                seen[i, ctx[r] + j] = True
                j = parents[start[r] + j]
        seen = seen.to(DEV)
        for h in range(case["hq"]):
            x = s["q"][start[r]:start[r] + int(m), h].double() @ k[:, h // rep].T / math.sqrt(case["d"])
            out[start[r]:start[r] + int(m), h] = torch.softmax(x.masked_fill(~seen, -math.inf), -1) @ v[:, h // rep]
    return out


def _exact_gdn(s, case, lens, start, parents):
    hk, hv, d, taps = case["hk"], case["hv"], case["d"], case["taps"]
    ids, accepted = s["ids"].tolist(), s["accepted"].tolist()
    if case["op"] == "conv_gate":
        x, w = s["x"].double(), s["w"].double()
        rows, windows = [], []
        for r, m in enumerate(lens):
            held = s["conv"][ids[r]].double()                    # [channels, taps - 1], the oldest first
            after = []
            for i in range(m):
                p = parents[start[r] + i]
                full = torch.cat([held if p < 0 else after[p], x[start[r] + i][:, None]], 1)
                after.append(full[:, 1:])
                rows.append((full * w).sum(1))
        y = torch.stack(rows)
        z = s["a"].double() + s["dt_bias"].double()
        g = -s["a_log"].double().exp() * torch.where(z > 20, z, (1 + z.exp()).log())
        return y / (1 + (-y).exp()), g, 1 / (1 + (-s["b"].double()).exp())
    rep = hv // hk
    unit = lambda t: t / (t.square().sum(-1, keepdim=True) + EPS).sqrt()
    q, k, v = unit(s["q"].double()) / math.sqrt(d), unit(s["k"].double()), s["v"].double()
    q, k = q.repeat_interleave(rep, 1), k.repeat_interleave(rep, 1)
    decay, beta = s["g"].double().exp(), s["beta"].double()

    def step(state, n):
        state = state * decay[n][:, None, None]
        change = beta[n][:, None] * (v[n] - torch.einsum("hkv,hk->hv", state, k[n]))
        return state + k[n][:, :, None] * change[:, None]

    if case["op"] == "commit":
        pool, conv = s["s_pool"].double(), s["conv_pool"].double()
        layer = case["layers"] - 1
        for r in range(len(lens)):
            path, i = [], accepted[r]
            while i >= 0:
                path.insert(0, int(start[r]) + i)
                i = parents[start[r] + i]
            state = pool[ids[r], layer]
            for n in path:
                state = step(state, n)
            pool[ids[r], layer] = state
            window = torch.cat([conv[ids[r], layer], s["x"][path].double().T], 1)
            conv[ids[r], layer] = window[:, window.shape[1] - (taps - 1):]
        return pool, conv
    out = torch.empty(s["n"], hv, d, dtype=torch.float64, device=DEV)
    for r, m in enumerate(lens):
        first, after = s["state"][ids[r]].double(), []
        for i in range(m):
            p, n = parents[start[r] + i], int(start[r]) + i
            after.append(step(first if p < 0 else after[p], n))
            out[n] = torch.einsum("hkv,hk->hv", after[-1], q[n])
    z = s["z"].double()
    return out / (out.square().mean(-1, keepdim=True) + EPS).sqrt() * s["norm_w"].double() * z / (1 + (-z).exp())
