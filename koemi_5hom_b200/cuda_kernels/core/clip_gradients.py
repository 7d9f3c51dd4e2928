"""Core front: the global gradient norm over many tensors, and clipping.

One launch sums the squares of every tensor, a second scales them; the tensors'
addresses travel in the kernels' parameters, so nothing is copied to the device
and nothing synchronises.
"""
from __future__ import annotations

from array import array
from typing import Iterable, Sequence

import torch
from torch import Tensor

from koemi_5hom_b200.cuda_kernels import _training
from koemi_5hom_b200.cuda_kernels.loader import CudaExtensionValidationError, load_cuda_extension

__all__ = ["clip_gradients", "gradient_norm"]

_CODES = {dtype: _training.DTYPE_CODES[dtype] for dtype in (torch.float32, torch.float16, torch.bfloat16)}


def clip_gradients(gradients: Iterable[Tensor], max_norm: float, *, out: Sequence[Tensor] | None = None) -> Tensor:
    """Scale ``gradients`` by ``min(1, max_norm / (norm + 1e-6))`` and return the norm before.

    ``norm`` is the 2-norm over all tensors (f32, bf16 and f16 may be mixed; any
    shapes, contiguous, one device), an fp32 scalar on their device. In place by
    default: nothing is written when the factor is one. With ``out`` (tensors of the same
    sizes and dtypes, not overlapping the gradients) the scaled values go there.
    A norm that is not finite gives the formula's result: zeros and NaNs for an
    infinite norm, NaNs for a NaN.
    """
    gradients = list(gradients)
    if isinstance(max_norm, bool) or not isinstance(max_norm, (int, float)) or not max_norm >= 0.0:
        raise CudaExtensionValidationError("max_norm must be a non-negative number")
    elements, codes = _table(gradients, "gradients")
    if out is None:
        out = gradients
    else:
        out = list(out)
        if _table(out, "out") != (elements, codes) or (out and out[0].device != gradients[0].device):
            raise CudaExtensionValidationError("out must match gradients in sizes, dtypes and device")
    return _run(gradients, out, elements, codes, float(max_norm))


def gradient_norm(gradients: Iterable[Tensor]) -> Tensor:
    """The 2-norm over all tensors, an fp32 scalar on their device (see :func:`clip_gradients`)."""
    gradients = list(gradients)
    return _run(gradients, None, *_table(gradients, "gradients"), 0.0)


def _run(gradients, out, elements, codes, max_norm: float) -> Tensor:
    if not gradients:
        raise CudaExtensionValidationError("gradients must not be empty")
    load_cuda_extension(device=gradients[0].device)
    with torch.no_grad():
        return _training.clip_gradients(gradients, out, elements, codes, max_norm)


def _table(tensors: list[Tensor], name: str) -> tuple[array, array]:
    """Element counts and dtype codes; the checks run as whole-list passes,
    which cost a third of a loop's statements per tensor."""
    if not all(isinstance(t, Tensor) for t in tensors):
        raise TypeError(f"{name} must be torch.Tensors")
    try:
        codes = array("i", map(_CODES.__getitem__, map(_training.attribute_dtype, tensors)))
    except KeyError as error:
        raise CudaExtensionValidationError(f"{name} must use float32, float16 or bfloat16; found {error.args[0]}") from None
    if not all(map(Tensor.is_contiguous, tensors)):
        raise CudaExtensionValidationError(f"{name} must be contiguous")
    devices = set(map(_training.attribute_device, tensors))
    if len(devices) > 1 or any(device.type != "cuda" for device in devices):
        raise CudaExtensionValidationError(f"{name} must be on one CUDA device, got {', '.join(sorted(map(str, devices)))}")
    return array("q", map(Tensor.numel, tensors)), codes
