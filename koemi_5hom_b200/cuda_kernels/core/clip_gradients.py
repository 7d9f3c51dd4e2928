"""Core front: the global gradient norm over many tensors, and clipping.

One launch sums the squares of every tensor, a second scales them; the tensors'
addresses travel in the kernels' parameters, so nothing is copied to the device
and nothing synchronises.
"""
from __future__ import annotations

from typing import Iterable, Sequence

import torch
from torch import Tensor

from koemi_5hom_b200 import _native
from koemi_5hom_b200.cuda_kernels import _training
from koemi_5hom_b200.cuda_kernels.loader import CudaExtensionValidationError, load_cuda_extension

__all__ = ["clip_gradients", "gradient_norm"]

_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def clip_gradients(gradients: Iterable[Tensor], max_norm: float, *, out: Sequence[Tensor] | None = None) -> Tensor:
    """Scale ``gradients`` by ``min(1, max_norm / (norm + 1e-6))`` and return the norm before.

    ``norm`` is the 2-norm over all tensors (f32, bf16 and f16 may be mixed; any
    shapes, contiguous, one device, none overlapping another), an fp32 scalar on their
    device. In place by default: nothing is written when the factor is one. With ``out``
    (tensors of the same sizes and dtypes, not overlapping the gradients) the scaled values
    go there. No derivative passes through it, and dispatch modes do not see it.
    A norm that is not finite gives the formula's result: zeros and NaNs for an
    infinite norm, NaNs for a NaN.
    """
    gradients = list(gradients)
    if isinstance(max_norm, bool) or not isinstance(max_norm, (int, float)) or not max_norm >= 0.0:
        raise CudaExtensionValidationError("max_norm must be a non-negative number")
    return _call(gradients, gradients if out is None else list(out), float(max_norm))


def gradient_norm(gradients: Iterable[Tensor]) -> Tensor:
    """The 2-norm over all tensors, an fp32 scalar on their device (see :func:`clip_gradients`)."""
    return _call(list(gradients), None, 0.0)


def _call(gradients: list, out: list | None, max_norm: float) -> Tensor:
    """The binding checks the tensors as it collects their addresses (a list of
    hundreds costs microseconds there); what it refuses is explained here."""
    lists = (gradients,) if out is None else (gradients, out)
    first = gradients[0] if gradients else None
    if not isinstance(first, Tensor) or not first.is_cuda:
        _explain(lists)
    if not _training.loaded():
        load_cuda_extension(device=first.device)
        _training.load(first.device)
    try:
        return _native.binding().koemi_torch_clip_gradients(gradients, out, max_norm)
    except (ValueError, TypeError, RuntimeError):
        _explain(lists)
        raise


def _explain(lists: tuple[list, ...]) -> None:
    """Raise the typed error for the first rule that the tensors break."""
    for name, tensors in zip(("gradients", "out"), lists):
        if not all(isinstance(t, Tensor) for t in tensors):
            raise TypeError(f"{name} must be torch.Tensors")
        if not tensors:
            raise CudaExtensionValidationError(f"{name} must not be empty")
        for t in tensors:
            if t.dtype not in _DTYPES:
                raise CudaExtensionValidationError(f"{name} must use float32, float16 or bfloat16; found {t.dtype}")
            if not t.is_contiguous():
                raise CudaExtensionValidationError(f"{name} must be contiguous")
        devices = {t.device for t in tensors}
        if len(devices) > 1 or next(iter(devices)).type != "cuda":
            raise CudaExtensionValidationError(f"{name} must be on one CUDA device, got {', '.join(sorted(map(str, devices)))}")
    if len(lists) == 2 and ([(t.numel(), t.dtype, t.device) for t in lists[0]] != [(t.numel(), t.dtype, t.device) for t in lists[1]]):
        raise CudaExtensionValidationError("out must match gradients in sizes, dtypes and device")
