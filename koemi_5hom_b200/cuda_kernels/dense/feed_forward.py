"""Dense front: the gated feed-forward block, forward and backward, on tensor cores.

The block that every expert of the routed MLP is
(src/koemi/model/experts.py:90-143), for rows that all take the same weights, with
its gradients. There is no CPU fallback.
"""
from __future__ import annotations

import torch
from torch import Tensor

from koemi_5hom_b200 import _native
from koemi_5hom_b200.cuda_kernels import _training
from koemi_5hom_b200.cuda_kernels.dense.affine_scan import (DenseCudaBuildError, DenseCudaUnavailableError,
                                                            DenseCudaValidationError, native_cuda_available)

__all__ = ["gated_feed_forward"]

_DTYPES = (torch.float16, torch.bfloat16, torch.float32)


def gated_feed_forward(values: Tensor, gate_weight: Tensor, value_weight: Tensor, output_weight: Tensor, *,
                       gate_bias: Tensor | None = None, value_bias: Tensor | None = None,
                       output_bias: Tensor | None = None) -> Tensor:
    """Return ``(silu(x Wg^T + bg) * (x Wv^T + bv)) Wo^T + bo`` for every row x of ``values``.

    ``values`` is ``[..., width]``, ``gate_weight`` and ``value_weight`` are
    ``[hidden, width]``, ``output_weight`` is ``[out, hidden]`` and the biases
    are ``[hidden]``, ``[hidden]``, ``[out]`` (zeros when omitted), all of one
    dtype: f32, bf16 or f16. Sums are fp32. In 16 bits the hidden values and
    their gradients are rounded to the type between the products: an fp16 hidden
    value past 65504 is infinite, and what a gradient of one has under 2^-14 loses
    digits, under 2^-25 everything, so scale an fp16 loss. fp32 products have fp32's
    precision, and an operand past 3.38e38 may give NaN. Differentiable to first order in everything; a call that may be
    differentiated keeps the hidden values, silu of the gate and the slope that the
    gate's gradient takes, 10 bytes a hidden value in 16 bits and 14 in fp32.
    """
    arguments = (values, gate_weight, value_weight, output_weight, gate_bias, value_bias, output_bias)
    if not _training.loaded():
        _validate(*arguments)
        try:
            _training.load(values.device)
        except _native.KoemiNativeUnavailableError as error:
            raise DenseCudaBuildError(f"failed to load the native dense CUDA library: {error}") from error
    try:
        return torch.ops.koemi_b200.gated_feed_forward.default(*arguments)
    except (ValueError, TypeError, RuntimeError):  # what the op refuses is explained here
        _validate(*arguments)
        raise


def _validate(values, gate_weight, value_weight, output_weight, gate_bias, value_bias, output_bias) -> None:
    def fail(message: str) -> None:
        raise DenseCudaValidationError(message)

    weights = (("gate_weight", gate_weight), ("value_weight", value_weight), ("output_weight", output_weight))
    biases = (("gate_bias", gate_bias), ("value_bias", value_bias), ("output_bias", output_bias))
    for name, tensor in (("values", values), *weights, *biases):
        if not isinstance(tensor, Tensor) and (tensor is not None or name not in dict(biases)):
            raise TypeError(f"{name} must be a torch.Tensor")
    if values.ndim < 1 or values.shape[-1] < 1:
        fail("values must have shape [..., width] with a positive width")
    if values.dtype not in _DTYPES:
        fail(f"unsupported CUDA dtype(s): {values.dtype}")
    width = values.shape[-1]
    if gate_weight.ndim != 2 or gate_weight.shape[1] != width or gate_weight.shape[0] < 1:
        fail(f"gate_weight must have shape [hidden, {width}], got {tuple(gate_weight.shape)}")
    hidden = gate_weight.shape[0]
    if value_weight.shape != gate_weight.shape:
        fail(f"value_weight must have shape {tuple(gate_weight.shape)}, got {tuple(value_weight.shape)}")
    if output_weight.ndim != 2 or output_weight.shape[1] != hidden or output_weight.shape[0] < 1:
        fail(f"output_weight must have shape [out, {hidden}], got {tuple(output_weight.shape)}")
    for (name, bias), size in zip(biases, (hidden, hidden, output_weight.shape[0])):
        if bias is not None and bias.shape != (size,):
            fail(f"{name} must have shape {(size,)}, got {tuple(bias.shape)}")
    for name, tensor in (*weights, *biases):
        if tensor is not None and tensor.dtype != values.dtype:
            fail(f"{name} must use the values' dtype {values.dtype}; found {tensor.dtype}")
    if not values.is_cuda and not native_cuda_available():
        raise DenseCudaUnavailableError("the native feed-forward block requires torch CUDA support, a CUDA device, and the built kernel library")
    for _, tensor in (("values", values), *weights, *biases):
        if tensor is not None and (not tensor.is_cuda or tensor.device != values.device):
            fail(f"all feed-forward tensors must use one CUDA device; found {values.device} and {tensor.device}")
