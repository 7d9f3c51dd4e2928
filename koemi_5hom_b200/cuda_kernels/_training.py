"""``torch.library`` ops of a training step over the C-ABI of ``libkoemi_b200.so``.

Same rules as ``_ops.py`` (outputs and workspace from torch's caching
allocator, launches on the current stream, fake implementations, no CPU
implementation), registered through ``torch.library.Library``: its dispatch
costs about 2 us a call where ``custom_op`` costs about 10, which counts for
operators whose kernels take a few microseconds. Gradients are defined by the
fronts' autograd functions, above these ops.
"""
from __future__ import annotations

from array import array
from contextlib import nullcontext
from operator import attrgetter

import torch
from torch import Tensor

from koemi_5hom_b200 import _native
from koemi_5hom_b200._native import DTYPE_CODES, ptr

_LIBRARY = torch.library.Library("koemi_b200", "FRAGMENT")
_HERE = nullcontext()
SEGMENT = 128  # positions between two carries of the gated recurrence


def _define(schema: str, implementation, fake):
    name = schema[:schema.index("(")]
    _LIBRARY.define(schema)
    _LIBRARY.impl(name, implementation, "CUDA")
    torch.library.register_fake(f"koemi_b200::{name}", fake, lib=_LIBRARY)
    return getattr(torch.ops.koemi_b200, name).default


def _on(device: torch.device):
    """A context in which ``device`` is current: the launches go to it."""
    _native.ensure_device(device)
    return _HERE if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _stream(device: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


def _run(function: str, *arguments) -> None:
    status = getattr(_native.library(), function)(*arguments)
    if status:
        _native.check(function, status)


# ------------------------------------------------------- the gated recurrence

def _gated_recurrence(projections, initial, valid, restart, low, high, keep):
    batch, length, double = projections.shape
    features = double // 2
    device = projections.device
    states = projections.new_empty((batch, length, features))
    final = torch.empty((batch, features), dtype=torch.float32, device=device)
    segments = -(-length // SEGMENT) if keep else 0
    carries = torch.empty((batch, segments, features), dtype=torch.float32, device=device)
    with _on(device):
        _run("koemi_dense_gated_recurrence_forward", projections.data_ptr(), ptr(initial), ptr(valid), ptr(restart),
             states.data_ptr(), final.data_ptr(), carries.data_ptr() if keep else None, batch, length, features, low,
             high, DTYPE_CODES[projections.dtype], _stream(device))
    return states, final, carries


def _gated_recurrence_fake(projections, initial, valid, restart, low, high, keep):
    batch, length, double = projections.shape
    f32 = dict(dtype=torch.float32)
    return (projections.new_empty((batch, length, double // 2)), projections.new_empty((batch, double // 2), **f32),
            projections.new_empty((batch, -(-length // SEGMENT) if keep else 0, double // 2), **f32))


gated_recurrence = _define(
    "gated_recurrence(Tensor projections, Tensor? initial, Tensor? valid, Tensor? restart, float low, float high, "
    "bool keep) -> (Tensor, Tensor, Tensor)", _gated_recurrence, _gated_recurrence_fake)


def _gated_recurrence_backward(projections, valid, restart, carries, grad_states, grad_final, low, high):
    batch, length, double = projections.shape
    device = projections.device
    grad_projections = torch.empty_like(projections)
    grad_initial = torch.empty((batch, double // 2), dtype=torch.float32, device=device)
    with _on(device):
        _run("koemi_dense_gated_recurrence_backward", projections.data_ptr(), ptr(valid), ptr(restart),
             carries.data_ptr(), ptr(grad_states), ptr(grad_final), grad_projections.data_ptr(),
             grad_initial.data_ptr(), batch, length, double // 2, low, high, DTYPE_CODES[projections.dtype],
             _stream(device))
    return grad_projections, grad_initial


gated_recurrence_backward = _define(
    "gated_recurrence_backward(Tensor projections, Tensor? valid, Tensor? restart, Tensor carries, "
    "Tensor? grad_states, Tensor? grad_final, float low, float high) -> (Tensor, Tensor)", _gated_recurrence_backward,
    lambda projections, valid, restart, carries, grad_states, grad_final, low, high: (
        torch.empty_like(projections),
        projections.new_empty((projections.shape[0], projections.shape[2] // 2), dtype=torch.float32)))


# ------------------------------------------------------------ the learned route

def _route_learned(logits, valid, top_k, renormalize):
    tokens, experts = logits.shape
    device = logits.device
    ids = torch.empty((tokens, top_k), dtype=torch.int64, device=device)
    weights = torch.empty((tokens, top_k), dtype=torch.float32, device=device)
    counts = torch.empty((experts,), dtype=torch.int64, device=device)
    balance = torch.empty((), dtype=torch.float32, device=device)
    slope = torch.empty((experts,), dtype=torch.float32, device=device)
    with _on(device):
        size = _native.library().koemi_moe_route_learned_workspace(tokens, experts)
        workspace = torch.empty(size, dtype=torch.uint8, device=device)
        _run("koemi_moe_route_learned_forward", logits.data_ptr(), ptr(valid), ids.data_ptr(), weights.data_ptr(),
             counts.data_ptr(), balance.data_ptr(), slope.data_ptr(), tokens, experts, top_k, renormalize,
             DTYPE_CODES[logits.dtype], workspace.data_ptr(), size, _stream(device))
    return ids, weights, counts, balance, slope


def _route_learned_fake(logits, valid, top_k, renormalize):
    tokens, experts = logits.shape
    f32 = dict(dtype=torch.float32)
    return (logits.new_empty((tokens, top_k), dtype=torch.int64), logits.new_empty((tokens, top_k), **f32),
            logits.new_empty((experts,), dtype=torch.int64), logits.new_empty((), **f32),
            logits.new_empty((experts,), **f32))


route_learned = _define(
    "route_learned(Tensor logits, Tensor? valid, int top_k, bool renormalize) -> "
    "(Tensor, Tensor, Tensor, Tensor, Tensor)", _route_learned, _route_learned_fake)


def _route_learned_backward(logits, ids, weights, slope, grad_weights, grad_balance, renormalize):
    tokens, experts = logits.shape
    device = logits.device
    grad = torch.empty_like(logits)
    with _on(device):
        _run("koemi_moe_route_learned_backward", logits.data_ptr(), ids.data_ptr(), weights.data_ptr(),
             ptr(grad_weights), ptr(grad_balance), slope.data_ptr(), grad.data_ptr(), tokens, experts, ids.shape[1],
             renormalize, DTYPE_CODES[logits.dtype], _stream(device))
    return grad


route_learned_backward = _define(
    "route_learned_backward(Tensor logits, Tensor ids, Tensor weights, Tensor slope, Tensor? grad_weights, "
    "Tensor? grad_balance, bool renormalize) -> Tensor", _route_learned_backward,
    lambda logits, ids, weights, slope, grad_weights, grad_balance, renormalize: torch.empty_like(logits))


# ------------------------------------------------------------- the policy loss

def _rows_of(logits: Tensor) -> tuple[int, int, int, int, int]:
    """rows, vocabulary, inner rows, outer stride, inner stride of [N, V] or [B, T, V] logits."""
    if logits.ndim == 2:
        return logits.shape[0], logits.shape[1], max(logits.shape[0], 1), 0, logits.stride(0)
    return (logits.shape[0] * logits.shape[1], logits.shape[2], max(logits.shape[1], 1), logits.stride(0),
            logits.stride(1))


def _policy_loss(logits, targets, old, advantages, reference, valid, clip_low, clip_high, kl_weight, with_gradient):
    rows = _rows_of(logits)
    device = logits.device
    loss, kl = torch.empty((), dtype=torch.float32, device=device), torch.empty((), dtype=torch.float32, device=device)
    log_probs = torch.empty(logits.shape[:-1], dtype=torch.float32, device=device)
    kept = torch.empty((2, rows[0]), dtype=torch.float32, device=device)  # lse | slopes
    gradient = torch.empty(logits.shape if with_gradient else (0,), dtype=logits.dtype, device=device)
    with _on(device):
        size = _native.library().koemi_think_policy_loss_workspace()
        workspace = torch.empty(size, dtype=torch.uint8, device=device)
        lse = kept.data_ptr()
        _run("koemi_think_policy_loss_forward", logits.data_ptr(), *rows, targets.data_ptr(), old.data_ptr(),
             advantages.data_ptr(), ptr(reference), ptr(valid), clip_low, clip_high, kl_weight, loss.data_ptr(),
             kl.data_ptr(), log_probs.data_ptr(), lse, lse + 4 * rows[0],
             gradient.data_ptr() if with_gradient else None, DTYPE_CODES[logits.dtype], workspace.data_ptr(), size,
             _stream(device))
    return loss, kl, log_probs, kept, gradient


def _policy_loss_fake(logits, targets, old, advantages, reference, valid, clip_low, clip_high, kl_weight, with_gradient):
    f32 = dict(dtype=torch.float32)
    return (logits.new_empty((), **f32), logits.new_empty((), **f32), logits.new_empty(logits.shape[:-1], **f32),
            logits.new_empty((2, _rows_of(logits)[0]), **f32), logits.new_empty(logits.shape if with_gradient else (0,)))


policy_loss = _define(
    "policy_loss(Tensor logits, Tensor targets, Tensor old, Tensor advantages, Tensor? reference, Tensor? valid, "
    "float clip_low, float clip_high, float kl_weight, bool with_gradient) -> (Tensor, Tensor, Tensor, Tensor, Tensor)",
    _policy_loss, _policy_loss_fake)


def _policy_loss_backward(logits, targets, valid, kept, grad_loss):
    rows = _rows_of(logits)
    device = logits.device
    grad = torch.empty(logits.shape, dtype=logits.dtype, device=device)
    lse = kept.data_ptr()
    with _on(device):
        _run("koemi_think_policy_loss_backward", logits.data_ptr(), *rows, targets.data_ptr(), ptr(valid), lse,
             lse + 4 * rows[0], grad_loss.data_ptr(), grad.data_ptr(), DTYPE_CODES[logits.dtype], _stream(device))
    return grad


policy_loss_backward = _define(
    "policy_loss_backward(Tensor logits, Tensor targets, Tensor? valid, Tensor kept, Tensor grad_loss) -> Tensor",
    _policy_loss_backward,
    lambda logits, targets, valid, kept, grad_loss: torch.empty(logits.shape, dtype=logits.dtype, device=logits.device))


def _policy_loss_scale(gradient, factor):
    with _on(gradient.device):
        _run("koemi_think_policy_loss_scale", gradient.data_ptr(), gradient.numel(), factor.data_ptr(),
             DTYPE_CODES[gradient.dtype], _stream(gradient.device))


policy_loss_scale = _define("policy_loss_scale(Tensor(a!) gradient, Tensor factor) -> ()", _policy_loss_scale,
                            lambda gradient, factor: None)


# ------------------------------------------------------ the clipping of gradients

def clip_gradients(gradients, outputs, elements: array, codes: array, max_norm: float) -> Tensor:
    """The norm; ``outputs`` (or None: norm only) receive the clipped values.
    Called without the dispatcher, which takes longer to convert two lists of
    hundreds of tensors than the kernels run."""
    device = gradients[0].device
    norm = torch.empty((), dtype=torch.float32, device=device)
    addresses = array("Q", map(Tensor.data_ptr, gradients))
    targets = addresses if outputs is gradients else None if outputs is None else array("Q", map(Tensor.data_ptr, outputs))
    sizes, count = elements.buffer_info()
    with _on(device):
        size = _native.library().koemi_core_clip_gradients_workspace(sizes, count)
        workspace = torch.empty(max(size, 4), dtype=torch.uint8, device=device)
        _run("koemi_core_clip_gradients", addresses.buffer_info()[0], None if targets is None else targets.buffer_info()[0],
             sizes, codes.buffer_info()[0], count, max_norm, norm.data_ptr(), workspace.data_ptr(), size, _stream(device))
    return norm


attribute_dtype, attribute_device = attrgetter("dtype"), attrgetter("device")
