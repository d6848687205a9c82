"""Which step a layer sees when it is installed into an engine that keeps its own per-step
context (no GPU needed)."""
import types

import pytest
import torch


class Engine:
    """A context module of the reference's shape: a new object at each set and reset."""

    def __init__(self):
        self.reset_context()

    def set_context(self, **kw):
        self.now = types.SimpleNamespace(**kw)

    def reset_context(self):
        self.now = types.SimpleNamespace()

    def get_context(self):
        return self.now


@pytest.fixture
def installed(pkg):
    """(engine, two layers of one model)"""
    engine, Q = Engine(), types.SimpleNamespace(Qwen3_5GatedDeltaNet=object)
    P = types.SimpleNamespace(get_tp_rank=lambda: 0, get_tp_size=lambda: 1, get_tp_group=lambda: None)
    cfg = types.SimpleNamespace(hidden_size=64, linear_num_key_heads=1, linear_num_value_heads=2,
                                linear_key_head_dim=64, linear_value_head_dim=64,
                                linear_conv_kernel_dim=4, rms_norm_eps=1e-6)
    previous = pkg.layer.install(Q, P, engine)
    yield engine, [Q.Qwen3_5GatedDeltaNet(cfg) for _ in range(2)]
    pkg.layer.uninstall(previous, Q)
    pkg.context.reset_context()


def drafts(pkg, nodes=3):
    cu, par = torch.tensor([0, nodes], dtype=torch.int32), torch.arange(nodes, dtype=torch.int32) - 1
    pkg.context.set_draft_context(cu, par, nodes, torch.zeros(1, dtype=torch.int64))
    return par


def test_drafts_reach_installed_layers(pkg, installed):
    engine, layers = installed
    engine.set_context(max_seqlen_q=1)
    for m in layers:
        assert m._get_context() is engine.now
    par = drafts(pkg)
    for m in layers:
        ctx = m._get_context()
        assert ctx.draft_parents is par and ctx.max_seqlen_q == 3


@pytest.mark.parametrize("end", ["set_context", "reset_context"])
def test_drafts_end_with_the_engine_s_step(pkg, installed, end):
    engine, layers = installed
    drafts(pkg)
    engine.set_context(max_seqlen_q=1)          # the engine's own part of the step may come after
    assert all(m._get_context().draft_parents is not None for m in layers)
    getattr(engine, end)()
    for m in layers:
        assert m._get_context() is engine.now
    assert pkg.context.get_context().linear_state_ids is None, "dropped"


def test_drafts_again_in_the_same_engine_step(pkg, installed):
    engine, layers = installed
    for nodes in (2, 5):
        par = drafts(pkg, nodes)
        assert all(m._get_context().draft_parents is par for m in layers)
    pkg.context.reset_context()
    assert layers[0]._get_context() is engine.now


def test_other_steps_of_this_package_do_not_reach_installed_layers(pkg, installed):
    engine, layers = installed
    pkg.context.set_context(max_seqlen_q=7)
    assert layers[0]._get_context() is engine.now
