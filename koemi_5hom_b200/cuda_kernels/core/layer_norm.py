"""Core front: layer norm, forward and backward.

One kernel reads every row once, forward; one more, backward, gives the values'
gradient and the reductions of the weight's and the bias's. There is no CPU
fallback.
"""
from __future__ import annotations

import math

import torch
from torch import Tensor

from koemi_5hom_b200.cuda_kernels import _training
from koemi_5hom_b200.cuda_kernels.loader import CudaExtensionValidationError, load_cuda_extension

__all__ = ["layer_norm"]

_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def layer_norm(values: Tensor, weight: Tensor, bias: Tensor | None = None, eps: float = 1e-5) -> Tensor:
    """Return ``(values - mean) / sqrt(variance + eps) * weight + bias`` over the last dimension.

    ``values`` is ``[..., width]`` (f32, bf16 or f16; rows of any stride);
    ``weight`` and ``bias`` are ``[width]``, both in the values' dtype or both
    in fp32. Statistics and sums are fp32: a row whose sum, or whose sum of
    squared distances from the mean, leaves fp32's range is not what the formula
    gives. The result has the values' dtype and is rounded once. Differentiable
    to first order in all three; the gradients of ``weight`` and ``bias`` are sums
    over all rows in a fixed order.
    """
    if not _training.loaded():
        _validate(values, weight, bias, eps)
        load_cuda_extension(device=values.device)
        _training.load(values.device)
    try:
        if values.ndim in (2, 3):
            return torch.ops.koemi_b200.layer_norm.default(values, weight, bias, eps)
        rows = values.reshape(-1, values.shape[-1])
        return torch.ops.koemi_b200.layer_norm.default(rows, weight, bias, eps).reshape(values.shape)
    except (ValueError, TypeError, RuntimeError, AttributeError, IndexError):  # what the op refuses is explained here
        _validate(values, weight, bias, eps)
        raise


def _validate(values, weight, bias, eps) -> None:
    def fail(message: str) -> None:
        raise CudaExtensionValidationError(message)

    for name, value in (("values", values), ("weight", weight), ("bias", bias)):
        if not isinstance(value, Tensor) and (value is not None or name != "bias"):
            raise TypeError(f"{name} must be a torch.Tensor")
    if values.ndim < 1 or values.shape[-1] < 1:
        fail("values must have shape [..., width] with a positive width")
    if values.dtype not in _DTYPES:
        fail(f"values must use float32, float16 or bfloat16; found {values.dtype}")
    width = values.shape[-1]
    for name, value in (("weight", weight), ("bias", bias)):
        if value is not None and value.shape != (width,):
            fail(f"{name} must have shape {(width,)}, got {tuple(value.shape)}")
        if value is not None and value.dtype not in (values.dtype, torch.float32):
            fail(f"{name} must use {values.dtype} or float32; found {value.dtype}")
    if bias is not None and bias.dtype != weight.dtype:
        fail(f"weight and bias must have the same dtype; found {weight.dtype} and {bias.dtype}")
    if isinstance(eps, bool) or not isinstance(eps, (int, float)) or not 0.0 <= eps <= 3e38 or math.isnan(eps):
        fail("eps must be a finite non-negative number")
    for value in (values, weight, bias):
        if value is not None and (not value.is_cuda or value.device != values.device):
            fail(f"all layer norm tensors must use one CUDA device; found {values.device} and {value.device}")
