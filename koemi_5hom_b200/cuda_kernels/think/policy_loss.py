"""Think front: clipped policy loss with a KL term over the head's logits.

``policy_loss`` scores the sampled tokens under the current logits and returns
the clipped surrogate loss, the mean KL estimate and the tokens' log-probs.
The gradient with respect to the logits is formed in the forward's own pass,
while a row is on chip (f32, bf16); f16 gradients, which underflow before the
factor of a scaled loss, are formed in the backward from the rows' kept maxima and sums.
"""
from __future__ import annotations

import ctypes
import math
from typing import NamedTuple

import torch
from torch import Tensor

from koemi_5hom_b200 import _native
from koemi_5hom_b200.cuda_kernels import _training
from koemi_5hom_b200.cuda_kernels.think.surprise import CudaThinkUnavailableError, CudaThinkValidationError

__all__ = ["PolicyLoss", "policy_loss"]

_DTYPES = (torch.float16, torch.bfloat16, torch.float32)


class PolicyLoss(NamedTuple):
    """``loss`` (fp32 scalar, differentiable), ``kl`` (fp32 scalar) and
    ``log_probs`` (fp32, the targets' shape), the last two without gradient."""

    loss: Tensor
    kl: Tensor
    log_probs: Tensor


def policy_loss(logits: Tensor, target_ids: Tensor, old_log_probs: Tensor, advantages: Tensor, *,
                reference_log_probs: Tensor | None = None, valid_mask: Tensor | None = None, clip_low: float = 0.2,
                clip_high: float = 0.2, kl_weight: float = 0.0) -> PolicyLoss:
    """Mean over valid positions of ``-min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_weight * kl``.

    ``r = exp(lp - old)`` with ``lp`` the target's log-softmax, and ``kl =
    exp(d) - d - 1`` with ``d = reference - lp`` (zero without reference).
    ``logits`` is ``[rows, V]`` or ``[batch, length, V]`` (f32, bf16 or f16;
    strided views such as ``logits[:, :-1]`` are read in place); the other
    tensors have its leading shape: int64 targets, fp32 log-probs and
    advantages, a bool mask. Positions that are not valid are not read, have
    log-prob 0 and gradient 0; with none valid the loss is 0. A target outside
    ``[0, V)`` at a valid position makes its log-prob, the loss and its row's gradient NaN.
    Differentiable to first order in ``logits``; while gradients are enabled
    for f32 and bf16 logits the call allocates the logits' gradient.
    """
    arguments = (logits, target_ids, old_log_probs, advantages, reference_log_probs, valid_mask, clip_low, clip_high, kl_weight)
    if not _training.loaded():
        _validate(*arguments)
        try:
            _training.load(logits.device)
        except _native.KoemiNativeUnavailableError as error:
            raise CudaThinkUnavailableError(str(error)) from error
    try:
        return PolicyLoss(*torch.ops.koemi_b200.policy_loss.default(*arguments))
    except (ValueError, TypeError, RuntimeError):  # what the op refuses is explained here
        _validate(*arguments)
        raise


def _validate(logits, targets, old, advantages, reference, valid, clip_low, clip_high, kl_weight) -> None:
    def fail(message: str) -> None:
        raise CudaThinkValidationError(message)

    named = (("logits", logits, None), ("target_ids", targets, torch.int64), ("old_log_probs", old, torch.float32),
             ("advantages", advantages, torch.float32), ("reference_log_probs", reference, torch.float32),
             ("valid_mask", valid, torch.bool))
    for name, value, _ in named:
        if not isinstance(value, Tensor) and (value is not None or name not in ("reference_log_probs", "valid_mask")):
            fail(f"{name} must be a torch.Tensor")
    if logits.ndim not in (2, 3) or logits.shape[-1] < 1:
        fail("logits must have shape [rows, vocabulary] or [batch, length, vocabulary]")
    if logits.dtype not in _DTYPES:
        fail("logits dtype must be float16, bfloat16 or float32")
    shape = logits.shape[:-1]
    for name, value, dtype in named[1:]:
        if value is not None and (value.shape != shape or value.dtype != dtype):
            fail(f"{name} must be {dtype} with shape {tuple(shape)}, got {value.dtype} {tuple(value.shape)}")
    if not (clip_low >= 0.0 and clip_high >= 0.0 and math.isfinite(ctypes.c_float(kl_weight).value)):
        fail("clip widths must be non-negative and kl_weight finite in fp32")
    if kl_weight != 0.0 and reference is None:
        fail("kl_weight needs reference_log_probs")
    if not logits.is_cuda and not torch.cuda.is_available():
        raise CudaThinkUnavailableError("native think CUDA kernel is unavailable: torch.cuda.is_available() is False")
    device = logits.device
    for name, value, _ in named:
        if value is not None and (not value.is_cuda or value.device != device):
            fail(f"all think tensors must be on one CUDA device; {name} is on {value.device}")
