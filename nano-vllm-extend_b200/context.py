"""Per-step context, mirroring the reference's nanovllm/utils/context.py.

The GDN layer reads ``cu_seqlens_q``, ``max_seqlen_q``, ``linear_state_ids``
and ``lens_q`` from it (qwen3_5.py:869-881).  The dataclass keeps every field
of the reference's Context, in the same order, so ``set_context`` calls
written for the reference work unchanged.  When the layer is installed into
the reference engine (:func:`layer.install`), it reads the engine's own
context instead of this one, but for steps of drafted trees, which the engine's
context has no place for: see :func:`step_context`.
"""
from __future__ import annotations

from dataclasses import dataclass, field

import torch


@dataclass(slots=True)
class Context:
    cu_seqlens_q: torch.Tensor | None = None
    cu_seqlens_k: torch.Tensor | None = None
    max_seqlen_q: int = 0
    max_seqlen_k: int = 0
    slot_mapping: torch.Tensor | None = None
    block_tables: torch.Tensor | None = None
    num_decode_tokens: int = 0
    flashinfer_decode: object | None = None
    flashinfer_prefill: object | None = None
    draft_slot_mapping: torch.Tensor | None = None
    draft_block_tables: torch.Tensor | None = None
    # per-sequence recurrent-state slot ids, int64 [bs] on the device
    linear_state_ids: torch.Tensor | None = None
    # host copy of the per-sequence query lengths (avoids a device sync)
    lens_q: list[int] | None = None
    vision_embeds: tuple = ()


@dataclass(slots=True)
class DraftContext(Context):
    """A step whose rows are drafted trees (not in the reference): sequence r owns the
    rows of cu_seqlens_q, at most max_seqlen_q of them, ``draft_parents`` (int32 [rows]
    on the device) holds each row's parent within its sequence, -1 for a row that
    follows the stored context.  The layers leave their slots' state as it is until the
    accepted paths are committed (layer.commit_drafts)."""
    draft_parents: torch.Tensor | None = None
    # the engine's context when an installed layer first read this one
    engine: object | None = field(default=None, repr=False, compare=False)


_CONTEXT = Context()


def get_context() -> Context:
    return _CONTEXT


def set_context(cu_seqlens_q=None, cu_seqlens_k=None, max_seqlen_q=0, max_seqlen_k=0,
                slot_mapping=None, block_tables=None, num_decode_tokens=0,
                flashinfer_decode=None, flashinfer_prefill=None,
                draft_slot_mapping=None, draft_block_tables=None,
                linear_state_ids=None, lens_q=None, vision_embeds=()):
    global _CONTEXT
    _CONTEXT = Context(cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k,
                       slot_mapping, block_tables, num_decode_tokens,
                       flashinfer_decode, flashinfer_prefill,
                       draft_slot_mapping, draft_block_tables,
                       linear_state_ids, lens_q, vision_embeds)


def set_draft_context(cu_seqlens, draft_parents, max_nodes, linear_state_ids):
    """Make the step one of drafted trees (:class:`DraftContext`), for layers installed
    into an engine too.  The tensors are read again when the accepted paths are committed,
    so they keep their contents until then."""
    global _CONTEXT
    _CONTEXT = DraftContext(cu_seqlens, cu_seqlens, max_nodes, max_nodes,
                            linear_state_ids=linear_state_ids, draft_parents=draft_parents)


def reset_context():
    global _CONTEXT
    _CONTEXT = Context()


def step_context(engine_context):
    """The step's context for a layer installed into an engine whose own one is
    ``engine_context()``: the drafted trees of :func:`set_draft_context` where these are
    set, else the engine's.  An engine never resets this module's context, so a step of
    drafted trees lasts until the engine sets or resets its own, at the latest: from the
    first layer's read on it belongs to the engine's context of that moment, and is
    dropped once that is another object, as each ``set_context`` and ``reset_context``
    makes one (an engine that changes its context in place calls this module's
    :func:`reset_context` after the step)."""
    own, step = _CONTEXT, engine_context()
    if not isinstance(own, DraftContext):
        return step
    if own.engine is None:
        own.engine = step
    if own.engine is step:
        return own
    reset_context()
    return step
