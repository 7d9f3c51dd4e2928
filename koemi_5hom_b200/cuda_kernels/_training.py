"""The training operators' dispatcher ops: loading them, and their fake implementations.

The ops (schemas, CUDA implementations, autograd formulas) live in C++, in
``lib/libkoemi_b200_torch.so`` (csrc/binding/training_ops.cpp), so that neither a
call nor a backward pass on autograd's thread runs Python; their outputs and
workspaces come from torch's caching allocator and their kernels run on the
current stream, as those of ``_ops.py``. There is no CPU implementation: the
fronts report CPU tensors before dispatch.
"""
from __future__ import annotations

import threading

import torch

from koemi_5hom_b200 import _native

SEGMENT = 128  # positions between two carries of the gated recurrence
_LOCK = threading.Lock()
_loaded = False


def register() -> None:
    """Register the ops and their fake implementations (once, whichever threads call first)."""
    global _loaded
    with _LOCK:
        if not _loaded:
            _native.binding()
            _register_fakes()
            _loaded = True


def load(device: torch.device) -> None:
    """Register the ops and initialise ``device``."""
    register()
    _native.ensure_device(device)


def loaded() -> bool:
    """Whether the ops are registered. They check their arguments and initialise their device themselves."""
    return _loaded


def _register_fakes() -> None:
    f32 = dict(dtype=torch.float32)

    def fake(name):
        return torch.library.register_fake(f"koemi_b200::{name}")

    @fake("gated_recurrence")
    def _(projections, initial, valid, restart, low, high):
        batch, length, double = projections.shape
        return projections.new_empty((batch, length, double // 2)), projections.new_empty((batch, double // 2), **f32)

    @fake("gated_recurrence_keep")
    def _(projections, initial, valid, restart, low, high):
        batch, length, double = projections.shape
        return (projections.new_empty((batch, length, double // 2)), projections.new_empty((batch, double // 2), **f32),
                projections.new_empty((batch, (length + SEGMENT - 1) // SEGMENT, double // 2), **f32))

    @fake("gated_recurrence_backward")
    def _(projections, valid, restart, carries, grad_states, grad_final, low, high):
        return (torch.empty_like(projections),
                projections.new_empty((projections.shape[0], projections.shape[2] // 2), **f32))

    def route(logits, top_k):
        tokens, experts = logits.shape
        return (logits.new_empty((tokens, top_k), dtype=torch.int64), logits.new_empty((tokens, top_k), **f32),
                logits.new_empty((experts,), dtype=torch.int64), logits.new_empty((), **f32))

    @fake("route_learned")
    def _(logits, valid, top_k, renormalize):
        return route(logits, top_k)

    @fake("route_learned_keep")
    def _(logits, valid, top_k, renormalize):
        return (*route(logits, top_k), logits.new_empty((logits.shape[1],), **f32))

    @fake("route_learned_backward")
    def _(logits, ids, weights, slope, grad_weights, grad_balance, renormalize):
        return torch.empty_like(logits)

    def policy(logits):
        return logits.new_empty((), **f32), logits.new_empty((), **f32), logits.new_empty(logits.shape[:-1], **f32)

    @fake("policy_loss")
    def _(logits, targets, old, advantages, reference, valid, clip_low, clip_high, kl_weight):
        return policy(logits)

    @fake("policy_loss_keep")
    def _(logits, targets, old, advantages, reference, valid, clip_low, clip_high, kl_weight):
        rows = logits.numel() // logits.shape[-1]
        at_once = logits.dtype != torch.float16
        return (*policy(logits), logits.new_empty((3, rows), **f32), logits.new_empty(logits.shape if at_once else (0,)))

    @fake("policy_loss_backward")
    def _(logits, targets, valid, kept, grad_loss):
        return logits.new_empty(logits.shape)

    @fake("policy_loss_scale")
    def _(gradient, factor):
        return None

    @fake("policy_loss_rescale")
    def _(gradient, logits, targets, valid, kept, factor):
        return None
