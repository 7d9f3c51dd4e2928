"""Dense front: the gated linear recurrence of a HERM block from raw projections.

``gated_recurrence`` takes the gate GEMM's output (retention | candidate, the
packed layout of ``gates_weight``) and runs the bounded gates
(src/koemi/model/memory.py:22-26), the padding masks, the restarts of packed
documents and the affine scan (model/scan.py:17-30) in one kernel, forward and
backward. There is no CPU fallback.
"""
from __future__ import annotations

import ctypes

import torch
from torch import Tensor

from koemi_5hom_b200 import _native
from koemi_5hom_b200.cuda_kernels import _training
from koemi_5hom_b200.cuda_kernels.dense.affine_scan import (DenseCudaBuildError, DenseCudaUnavailableError,
                                                            DenseCudaValidationError, native_cuda_available)

__all__ = ["gated_recurrence"]

_DTYPES = (torch.float16, torch.bfloat16, torch.float32)


def gated_recurrence(projections: Tensor, initial: Tensor | None = None, *, valid: Tensor | None = None,
                     restart: Tensor | None = None, minimum_retention: float = 2.0 ** -8,
                     maximum_retention: float = 1.0 - 2.0 ** -8) -> tuple[Tensor, Tensor]:
    """Run ``h_t = a_t h' + (1 - a_t) tanh(c_t)`` and return (states, final state).

    ``projections`` is ``[batch, length, 2 F]`` (p | c; f32, bf16 or f16) and
    ``a = minimum + (maximum - minimum) sigmoid(p)``; ``h'`` is ``h_{t-1}``, or
    zero where ``restart`` (bool ``[batch, length]``: the first position of a
    packed document). A position where ``valid`` (same shape) is false keeps
    the state, whatever its projections hold. ``initial`` is fp32 ``[batch, F]``
    (zeros when omitted). States have the projections' dtype; the running state
    and the returned final state are fp32. Differentiable to first order in
    ``projections`` and ``initial``; a single token is ``length == 1``.
    """
    if not _training.loaded():
        _validate(projections, initial, valid, restart, minimum_retention, maximum_retention)
        try:
            _training.load(projections.device)
        except _native.KoemiNativeUnavailableError as error:
            raise DenseCudaBuildError(f"failed to load the native dense CUDA library: {error}") from error
    try:
        return torch.ops.koemi_b200.gated_recurrence.default(projections, initial, valid, restart, minimum_retention,
                                                             maximum_retention)
    except (ValueError, TypeError, RuntimeError):  # what the op refuses is explained here
        _validate(projections, initial, valid, restart, minimum_retention, maximum_retention)
        raise


def _validate(projections, initial, valid, restart, low, high) -> None:
    def fail(message: str) -> None:
        raise DenseCudaValidationError(message)

    for name, value in (("projections", projections), ("initial", initial), ("valid", valid), ("restart", restart)):
        if not isinstance(value, Tensor) and (value is not None or name == "projections"):
            raise TypeError(f"{name} must be a torch.Tensor")
    if projections.ndim != 3 or projections.shape[2] % 2:
        fail("projections must have shape [batch, length, 2 * features]")
    if projections.dtype not in _DTYPES:
        fail(f"unsupported CUDA dtype(s): {projections.dtype}")
    batch, length, double = projections.shape
    if initial is not None and (initial.shape != (batch, double // 2) or initial.dtype != torch.float32):
        fail(f"initial must be float32 with shape {(batch, double // 2)}, got {initial.dtype} {tuple(initial.shape)}")
    for name, mask in (("valid", valid), ("restart", restart)):
        if mask is not None and (mask.shape != (batch, length) or mask.dtype != torch.bool):
            fail(f"{name} must be bool with shape {(batch, length)}, got {mask.dtype} {tuple(mask.shape)}")
    if not (0.0 < ctypes.c_float(low).value and low <= high and ctypes.c_float(high).value < 1.0):
        fail("retention bounds must satisfy 0 < minimum <= maximum < 1 in fp32")
    if not projections.is_cuda and not native_cuda_available():
        raise DenseCudaUnavailableError("native gated recurrence requires torch CUDA support, a CUDA device, and the built kernel library")
    for value in (projections, initial, valid, restart):
        if value is not None and (not value.is_cuda or value.device != projections.device):
            fail(f"all recurrence tensors must use one CUDA device; found {projections.device} and {value.device}")
