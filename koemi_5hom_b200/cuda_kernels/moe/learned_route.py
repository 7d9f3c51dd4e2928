"""MoE front: the learned route of a training step, with its balance loss and gradients.

``route_learned_topk`` is the reference's learned gate (src/koemi/model/router.py:43-59)
as one operator: softmax over the gate's logits, top-k, per-expert counts and
the balance loss of ``RouterStatistics``, differentiable in the logits through
the weights and the loss.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch import Tensor

from koemi_5hom_b200 import _native
from koemi_5hom_b200.cuda_kernels import _training

__all__ = ["LearnedRoute", "route_learned_topk"]

_DTYPES = (torch.float32, torch.float16, torch.bfloat16)
_EXPERT_LIMIT, _TOP_K_LIMIT = 4096, 256


class LearnedRoute(NamedTuple):
    """``expert_ids`` [tokens, k] int64, ``weights`` [tokens, k] fp32, ``counts``
    [experts] int64 and ``balance_loss`` (fp32 scalar)."""

    expert_ids: Tensor
    weights: Tensor
    counts: Tensor
    balance_loss: Tensor


def route_learned_topk(gate_logits: Tensor, valid_mask: Tensor | None = None, *, top_k: int,
                       renormalize: bool = False) -> LearnedRoute:
    """Choose the ``top_k`` largest logits of every row (ties: lowest expert id).

    ``gate_logits`` is ``[tokens, experts]`` (f32, bf16 or f16; at most 4096
    experts). Weights are softmax probabilities, divided by their sum when
    ``renormalize``. The balance loss is ``E sum_e importance_e load_e``:
    importance the mean probability over the rows that take part, load the
    share of the pairs (no gradient through the counts). Rows where
    ``valid_mask`` is false, and rows whose logits are all -inf, take no part:
    ids -1, weights and gradient zero. A NaN logit is never preferred and makes
    its row's weights NaN. Differentiable to first order in the logits.
    """
    if not _training.loaded():
        _validate(gate_logits, valid_mask, top_k)
        try:
            _training.load(gate_logits.device)
        except _native.KoemiNativeUnavailableError as error:
            from koemi_5hom_b200.cuda_kernels.moe import CudaMoeUnavailableError  # the package imports this module
            raise CudaMoeUnavailableError(f"Koemi MoE CUDA library failed to load: {error}") from error
    try:
        if type(top_k) is not int:  # the dispatcher takes bools
            raise TypeError("top_k must be an integer")
        return LearnedRoute(*torch.ops.koemi_b200.route_learned.default(gate_logits, valid_mask, top_k, bool(renormalize)))
    except (ValueError, TypeError, RuntimeError):  # what the op refuses is explained here
        _validate(gate_logits, valid_mask, top_k)
        raise


def _validate(gate_logits, valid_mask, top_k) -> None:
    from koemi_5hom_b200.cuda_kernels.moe import CudaMoeValidationError  # the package imports this module

    def fail(message: str) -> None:
        raise CudaMoeValidationError(message)

    for name, value in (("gate_logits", gate_logits), ("valid_mask", valid_mask)):
        if not isinstance(value, Tensor) and (value is not None or name == "gate_logits"):
            raise TypeError(f"{name} must be a torch.Tensor")
    if gate_logits.ndim != 2 or gate_logits.shape[1] < 1:
        fail("gate_logits must have shape [tokens, experts]")
    if gate_logits.dtype not in _DTYPES:
        fail(f"gate_logits must use float32, float16, or bfloat16; found {gate_logits.dtype}")
    tokens, experts = gate_logits.shape
    if experts > _EXPERT_LIMIT:
        fail(f"expert_count exceeds the learned route's limit of {_EXPERT_LIMIT}")
    if type(top_k) is not int or not 1 <= top_k <= min(experts, _TOP_K_LIMIT):
        fail(f"top_k must be an integer in [1, min(experts, {_TOP_K_LIMIT})]")
    if valid_mask is not None and (valid_mask.shape != (tokens,) or valid_mask.dtype != torch.bool):
        fail("valid_mask must be boolean with shape [tokens]")
    if not gate_logits.is_cuda or (valid_mask is not None and valid_mask.device != gate_logits.device):
        fail("gate_logits and valid_mask must be CUDA tensors on one device")
