"""A layer installed into an engine's modules checks drafted trees and commits them: the same
bits as a layer of this package on its own, and pools that the check does not touch."""
import types

import numpy as np
import pytest
import torch

import _tree_reference as R
from test_gpu_tree import i32, i64
from test_gpu_tree_layer import DEV, forward, make_layer, pkg_gpu  # noqa: F401
from test_tree_context import Engine

pytestmark = pytest.mark.gpu


def test_an_installed_layer_checks_a_tree_and_commits(pkg_gpu, monkeypatch):  # noqa: F811
    pkg, engine = pkg_gpu, Engine()
    Q = types.SimpleNamespace(Qwen3_5GatedDeltaNet=object)
    P = types.SimpleNamespace(get_tp_rank=lambda: 0, get_tp_size=lambda: 1, get_tp_group=lambda: None)
    own = make_layer(pkg, 128, seed=4)
    previous = pkg.layer.install(Q, P, engine)
    try:
        plain = pkg.layer.Qwen3_5GatedDeltaNet
        monkeypatch.setattr(pkg.layer, "Qwen3_5GatedDeltaNet", Q.Qwen3_5GatedDeltaNet)
        inst = make_layer(pkg, 128, seed=4)
        monkeypatch.setattr(pkg.layer, "Qwen3_5GatedDeltaNet", plain)
    finally:
        pkg.layer.uninstall(previous, Q)
    lens, ids, g = [7, 0, 12], i64([4, 0, 2]), torch.Generator(device=DEV).manual_seed(1)
    par, x = i32(np.concatenate(R.make_trees(lens, 3))), torch.randn(19, 256, generator=g, device=DEV)
    x, pools = x.to(torch.bfloat16), []
    for m in (own, inst):
        p = pkg.state_pool.StatePools([m], 6, DEV)
        p.s_pool.normal_(0, 0.1, generator=g.manual_seed(2))
        p.conv_pool.normal_(0, 1, generator=g.manual_seed(3))
        pools.append(p)
    want = forward(pkg, own, x, ids, lens, par)
    before = [pools[1].s_pool.clone(), pools[1].conv_pool.clone()]
    # the engine's step as it stands from before: 19 decode rows, which would move 19 states
    engine.set_context(cu_seqlens_q=None, max_seqlen_q=1, linear_state_ids=i64([4] * 19), lens_q=None)
    pkg.context.set_draft_context(i32(R.cu_of(lens)), par, 12, ids)
    with torch.inference_mode():
        got = inst(None, x)
    assert torch.equal(got, want)
    assert torch.equal(pools[1].s_pool, before[0]) and torch.equal(pools[1].conv_pool, before[1])
    acc = i32([6, -1, 9])
    own.commit_drafts(acc)
    pkg.layer.commit_drafts(torch.nn.ModuleList([inst]), acc)
    assert torch.equal(pools[0].s_pool, pools[1].s_pool) and torch.equal(pools[0].conv_pool, pools[1].conv_pool)
    assert not torch.equal(pools[1].s_pool, before[0])
    # the engine's next step is its own again
    step = dict(cu_seqlens_q=None, max_seqlen_q=1, linear_state_ids=ids, lens_q=None)
    engine.set_context(**step)
    with torch.inference_mode():
        got = inst(None, x[:3])
    with pytest.raises(RuntimeError, match="no drafted rows"):
        inst.commit_drafts(acc)
    assert torch.equal(got, forward(pkg, own, x[:3], ids, [1, 1, 1]))
    assert torch.equal(pools[0].s_pool, pools[1].s_pool)
    assert pkg.ops.check_status() == 0
