"""Core front: dropout from a counter-based generator, with an optional residual.

The mask is a function of (seed, site, step, position) and is never stored: the
backward pass computes it again. There is no CPU fallback.
"""
from __future__ import annotations

import torch
from torch import Tensor

from koemi_5hom_b200.cuda_kernels import _training
from koemi_5hom_b200.cuda_kernels.loader import CudaExtensionValidationError, load_cuda_extension

__all__ = ["dropout"]

_DTYPES = (torch.float32, torch.float16, torch.bfloat16)
_WORD = 1 << 64


def dropout(values: Tensor, probability: float, *, seed: int, site: int = 0, step: int | Tensor = 0,
            residual: Tensor | None = None) -> Tensor:
    """Return ``residual + where(kept, values / (1 - probability), 0)``.

    ``values`` is f32, bf16 or f16 of any shape, ``residual`` (zeros when
    omitted) of the same shape and dtype. The probability is taken to the
    nearest multiple of 2^-16, and the scale is that multiple's, so the mean is
    kept exactly. Which values stay depends only on ``seed``, ``site`` (the
    place in the model), ``step`` (each in [0, 2^64)) and the position in
    row-major order; give every call of a step its own site, and every step its
    own number. A ``step`` on the device (a zero-dimensional int64 CUDA tensor)
    is read by the kernel, so that a captured graph draws new numbers when the
    program advances it; it must not change between a pass's forward and backward. A dropped
    value may be anything, infinities and NaN too. Differentiable in reverse mode.
    ``torch.vmap`` over it is refused: a position names its bits, so every sample
    would get the same mask.
    """
    if isinstance(probability, bool) or not isinstance(probability, (int, float)) or not 0.0 <= probability <= 1.0:
        raise CudaExtensionValidationError("probability must be in [0, 1]")
    on_device = isinstance(step, Tensor)
    for name, number in (("seed", seed), ("site", site), ("step", 0 if on_device else step)):
        if isinstance(number, bool) or not isinstance(number, int) or not 0 <= number < _WORD:
            raise CudaExtensionValidationError(f"{name} must be an integer in [0, 2^64)")
    if not _training.loaded():
        _validate(values, residual, step)
        load_cuda_extension(device=values.device)
        _training.load(values.device)
    try:
        return torch.ops.koemi_b200.dropout.default(values, residual, step if on_device else None, int(probability * 65536 + 0.5),
                                                    _signed(seed), _signed(site), 0 if on_device else _signed(step))
    except (ValueError, TypeError, RuntimeError):  # what the op refuses is explained here
        _validate(values, residual, step)
        raise


def _signed(number: int) -> int:
    """The op's 64-bit integers are signed."""
    return number - _WORD if number >> 63 else number


def _validate(values, residual, step) -> None:
    def fail(message: str) -> None:
        raise CudaExtensionValidationError(message)

    for name, value in (("values", values), ("residual", residual)):
        if not isinstance(value, Tensor) and (value is not None or name == "values"):
            raise TypeError(f"{name} must be a torch.Tensor")
    if values.dtype not in _DTYPES:
        fail(f"values must use float32, float16 or bfloat16; found {values.dtype}")
    if residual is not None and (residual.shape != values.shape or residual.dtype != values.dtype):
        fail(f"residual must match values in shape and dtype, got {residual.dtype} {tuple(residual.shape)}")
    if isinstance(step, Tensor) and (step.shape != () or step.dtype != torch.int64):
        fail(f"a step on the device must be a zero-dimensional int64 tensor, got {step.dtype} {tuple(step.shape)}")
    for value in (values, residual, step):
        if isinstance(value, Tensor) and (not value.is_cuda or value.device != values.device):
            fail(f"all dropout tensors must use one CUDA device; found {values.device} and {value.device}")
