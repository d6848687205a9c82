"""What the tree operators refuse before any launch, and the host-side tree
checks (no GPU needed: the C entry points return before they touch a pointer)."""
import pytest
import torch

FAKE = 1 << 20                      # aligned, never dereferenced


def _call(pkg, name, args):
    lib = pkg._lib.load()
    rc = getattr(lib, name)(*args.values())
    return rc, lib.gdn_last_error().decode()


def conv_args(**kw):
    a = dict(x=FAKE, xs=1024, pool=FAKE, ss=1024 * 3, slots=4, ids=FAKE, cu=FAKE, n_seqs=2,
             parents=FAKE, max_nodes=8, n=10, C=1024, K=4, w=FAKE, y=FAKE, ys=1024, b=FAKE, a=FAKE,
             abs_=8, H=8, a_log=FAKE, dt=FAKE, pdt=0, g=FAKE, beta=FAKE, status=None, stream=None)
    return {**a, **kw}


def delta_args(**kw):
    a = dict(q=FAKE, qs=512, k=FAKE, ks=512, v=FAKE, vs=1024, g=FAKE, beta=FAKE, pool=FAKE,
             ss=8 * 128 * 128, slots=4, ids=FAKE, cu=FAKE, n_seqs=2, parents=FAKE, max_nodes=8, n=10,
             out=FAKE, HK=4, HV=8, DK=128, DV=128, scale=0.1, z=None, zs=0, nw=None, eps=1e-6,
             status=None, stream=None)
    return {**a, **kw}


def commit_args(**kw):
    a = dict(x=FAKE, xs=2048, k=FAKE, ks=512, v=FAKE, vs=1024, g=FAKE, beta=FAKE, conv=FAKE,
             css=2048 * 3, C=2048, K=4, pool=FAKE, ss=8 * 128 * 128, slots=4, ids=FAKE, cu=FAKE,
             n_seqs=2, parents=FAKE, accepted=FAKE, max_nodes=8, n=10, HK=4, HV=8, DK=128, DV=128,
             status=None, stream=None)
    return {**a, **kw}


def rope_args(**kw):
    a = dict(q=FAKE, qs=2048, k=FAKE, ks=512, v=FAKE, vs=512, qw=FAKE, kw=FAKE, eps=1e-6, off=0,
             cs=FAKE, max_pos=100, rot=64, pos=FAKE, kc=FAKE, vc=FAKE, bs=256 * 512, ts=512, hs=128,
             blocks=8, block=256, slot=FAKE, out=FAKE, n=10, HQ=16, HKV=4, D=128, status=None,
             stream=None)
    return {**a, **kw}


def attn_args(**kw):
    a = dict(q=FAKE, qs=2048, kc=FAKE, vc=FAKE, bs=256 * 512, ts=512, hs=128, blocks=8, block=256,
             table=FAKE, tstride=16, max_blocks=16, ctx=FAKE, cu=FAKE, n_seqs=2, parents=FAKE,
             max_nodes=8, n=10, max_len=200, out=FAKE, HQ=16, HKV=4, D=128, scale=0.1, ws=None, wsb=0,
             status=None, stream=None)
    return {**a, **kw}


def slot_args(**kw):
    a = dict(table=FAKE, tstride=16, max_blocks=16, ctx=FAKE, cu=FAKE, n_seqs=2, parents=FAKE,
             accepted=None, max_nodes=8, block=256, n=10, pos=FAKE, slot=FAKE, status=None,
             stream=None)
    return {**a, **kw}


INVALID, UNSUPPORTED = 1, 2

REFUSED = [
    ("gdn_conv_gate_tree", conv_args, dict(max_nodes=65), UNSUPPORTED, "65 nodes"),
    ("gdn_conv_gate_tree", conv_args, dict(max_nodes=-1), INVALID, "max_nodes"),
    ("gdn_conv_gate_tree", conv_args, dict(K=5), UNSUPPORTED, "kernel"),
    ("gdn_conv_gate_tree", conv_args, dict(xs=1000), INVALID, "row stride"),
    ("gdn_conv_gate_tree", conv_args, dict(ss=100), INVALID, "slot_stride"),
    ("gdn_conv_gate_tree", conv_args, dict(abs_=4), INVALID, "row stride"),
    ("gdn_conv_gate_tree", conv_args, dict(pdt=3), INVALID, "param_dtype"),
    ("gdn_conv_gate_tree", conv_args, dict(parents=None), INVALID, "null"),
    ("gdn_delta_rule_tree", delta_args, dict(max_nodes=65), UNSUPPORTED, "65 nodes"),
    ("gdn_delta_rule_tree", delta_args, dict(DK=96, DV=96), UNSUPPORTED, "head dims"),
    ("gdn_delta_rule_tree", delta_args, dict(DK=64), UNSUPPORTED, "head dims"),
    ("gdn_delta_rule_tree", delta_args, dict(HK=3), INVALID, "multiple"),
    ("gdn_delta_rule_tree", delta_args, dict(ss=1000), INVALID, "slot_stride"),
    ("gdn_delta_rule_tree", delta_args, dict(vs=1000), INVALID, "row stride"),
    ("gdn_delta_rule_tree", delta_args, dict(z=FAKE, zs=1024), INVALID, "norm_weight"),
    ("gdn_delta_rule_tree", delta_args, dict(v=FAKE + 2), UNSUPPORTED, "aligned"),
    ("gdn_delta_rule_tree", delta_args, dict(pool=FAKE + 4), INVALID, "aligned"),
    ("gdn_delta_rule_tree", delta_args, dict(q=None), INVALID, "null"),
    ("gdn_commit_tree", commit_args, dict(max_nodes=100), UNSUPPORTED, "100 nodes"),
    ("gdn_commit_tree", commit_args, dict(accepted=None), INVALID, "null"),
    ("gdn_commit_tree", commit_args, dict(css=7), INVALID, "conv_slot_stride"),
    ("gdn_commit_tree", commit_args, dict(K=1), UNSUPPORTED, "kernel"),
    ("gdn_commit_tree", commit_args, dict(DK=32, DV=32), UNSUPPORTED, "head dims"),
    ("gdn_qk_norm_rope_cache", rope_args, dict(D=96), UNSUPPORTED, "head dim"),
    ("gdn_qk_norm_rope_cache", rope_args, dict(rot=24), UNSUPPORTED, "rotary"),
    ("gdn_qk_norm_rope_cache", rope_args, dict(rot=144), UNSUPPORTED, "rotary"),
    ("gdn_qk_norm_rope_cache", rope_args, dict(qs=100), INVALID, "row stride"),
    ("gdn_qk_norm_rope_cache", rope_args, dict(block=0), INVALID, "cache"),
    ("gdn_qk_norm_rope_cache", rope_args, dict(q=FAKE + 8), UNSUPPORTED, "aligned"),
    ("gdn_qk_norm_rope_cache", rope_args, dict(ts=513), UNSUPPORTED, "aligned"),
    ("gdn_qk_norm_rope_cache", rope_args, dict(slot=None), INVALID, "null"),
    ("gdn_attention_tree", attn_args, dict(max_nodes=65), UNSUPPORTED, "65 nodes"),
    ("gdn_attention_tree", attn_args, dict(D=80), UNSUPPORTED, "head dim"),
    ("gdn_attention_tree", attn_args, dict(HKV=3), INVALID, "multiple"),
    ("gdn_attention_tree", attn_args, dict(max_len=0), INVALID, "max_len"),
    ("gdn_attention_tree", attn_args, dict(), INVALID, "workspace"),
    ("gdn_attention_tree", attn_args, dict(scale=0.0), INVALID, "scale"),
    ("gdn_attention_tree", attn_args, dict(scale=float("nan")), INVALID, "scale"),
    ("gdn_attention_tree", attn_args, dict(max_len=1 << 29), UNSUPPORTED, "max_len"),
    ("gdn_attention_tree", attn_args, dict(blocks=0), INVALID, "pages"),
    ("gdn_attention_tree", attn_args, dict(hs=60), INVALID, "strides"),
    ("gdn_attention_tree", attn_args, dict(kc=FAKE + 2), UNSUPPORTED, "aligned"),
    ("gdn_attention_tree", attn_args, dict(table=None), INVALID, "null"),
    ("gdn_tree_slot_map", slot_args, dict(max_nodes=65), UNSUPPORTED, "65 nodes"),
    ("gdn_tree_slot_map", slot_args, dict(block=0), INVALID, "block"),
    ("gdn_tree_slot_map", slot_args, dict(tstride=8), INVALID, "block tables"),
    ("gdn_tree_slot_map", slot_args, dict(parents=None), INVALID, "null"),
]


@pytest.mark.parametrize("name,make,change,code,word", REFUSED)
def test_refusals(pkg, name, make, change, code, word):
    rc, msg = _call(pkg, name, make(**change))
    assert rc == code and word in msg and msg.startswith(name), msg


@pytest.mark.parametrize("name,make,change", [
    ("gdn_conv_gate_tree", conv_args, dict(n=0)), ("gdn_conv_gate_tree", conv_args, dict(n_seqs=0)),
    ("gdn_delta_rule_tree", delta_args, dict(n=0)), ("gdn_delta_rule_tree", delta_args, dict(n_seqs=0)),
    ("gdn_commit_tree", commit_args, dict(n_seqs=0)), ("gdn_qk_norm_rope_cache", rope_args, dict(n=0)),
    ("gdn_attention_tree", attn_args, dict(n=0)), ("gdn_attention_tree", attn_args, dict(n_seqs=0)),
    ("gdn_tree_slot_map", slot_args, dict(n=0))])
def test_empty_calls_are_noops(pkg, name, make, change):
    assert _call(pkg, name, make(**change))[0] == 0


def test_attention_workspace(pkg):
    """Two parts per CTA (148 SMs x 2, or x 1 for wide trees and head dim 256) of a row tile's fp32
    rows with maximum and sum, after the padded int64 tile counts."""
    f = pkg._lib.load().gdn_attention_tree_workspace_bytes
    assert f(0, 16, 4, 128, 1) == 0 and f(4, 16, 4, 128, 0) == 0
    assert f(8, 16, 4, 128, 1) == 256 + 296 * 2 * 16 * (4 * 128 + 8)
    assert f(31, 16, 4, 128, 17) == 256 + 148 * 2 * 128 * (4 * 128 + 8)
    assert f(32, 8, 4, 256, 16) == 512 + 148 * 2 * 32 * (4 * 256 + 8)


def test_cpu_tensors_are_refused(pkg):
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(AssertionError, match="CUDA"):
        pkg.ops.tree_slot_map(torch.zeros(2, 4, dtype=torch.int32), i[:2], i, i[:2], 1, 16, 2)
    with pytest.raises(AssertionError, match="CUDA"):
        pkg.ops.attention_tree(x.view(2, 1, 64), x, x, i, i, i, i, 1, 1)


def test_tree_checks(pkg):
    ops = pkg.ops
    cu, par = [0, 3, 3, 5], [-1, 0, 0, -1, -1]
    ops.check_tree(cu, par, 3, 5, accepted=[2, -1, 0])
    ops.check_tree(cu, par + [99, 99], 3, 7)              # rows behind the last sequence
    for bad in ([0, 3, 2, 5], [1, 3, 3, 5], [0, 3, 3, 6]):
        with pytest.raises(ValueError, match="cu_seqlens"):
            ops.check_tree(bad, par + [-1], 3, 5)
    with pytest.raises(ValueError, match="max_nodes"):
        ops.check_tree(cu, par, 2, 5)
    for bad in ([-1, 1, 0, -1, -1], [-1, 0, 0, -2, -1], [-1, 0, 0, 0, -1]):
        with pytest.raises(ValueError, match="parent"):
            ops.check_tree(cu, bad, 3, 5)
    for bad in ([3, -1, 0], [0, 0, 0], [0, -2, 0]):
        with pytest.raises(ValueError, match="accepted"):
            ops.check_tree(cu, par, 3, 5, accepted=bad)


@pytest.mark.parametrize("bit,error", [(0x8, ValueError), (0x10, IndexError)])
def test_status_bits_raise(pkg, bit, error):
    with pytest.raises(error):
        pkg.ops._raise_for(bit)
