"""Scalars that fp64 holds and the kernels' fp32 does not: refused by the fronts, in their own error types."""
from __future__ import annotations

import pytest
import torch

from koemi_5hom_b200.cuda_kernels import dense, think


@pytest.mark.parametrize("bounds", [(0.5, 1.0 - 1e-9), (1e-50, 0.5), (0.5, 0.5 - 1e-12), (1e-50, 1.0 - 1e-9)])
def test_retention_bounds_are_those_of_fp32(bounds):
    x = torch.zeros(2, 3, 8)
    low, high = bounds
    with pytest.raises(dense.DenseCudaValidationError, match="retention bounds"):
        dense.gated_recurrence(x, minimum_retention=low, maximum_retention=high)


def test_kl_weights_are_those_of_fp32():
    rows = torch.zeros(4)
    with pytest.raises(think.CudaThinkValidationError, match="kl_weight finite"):
        think.policy_loss(torch.zeros(4, 9), rows.long(), rows, rows, reference_log_probs=rows, kl_weight=1e39)


@pytest.mark.gpu
def test_scalars_are_refused_on_the_gpu(cuda):
    x, rows = torch.zeros(2, 3, 8, device=cuda), torch.zeros(4, device=cuda)
    dense.gated_recurrence(x)  # from here on the ops check first
    for low, high in ((0.5, 1.0 - 1e-9), (1e-50, 0.5), (0.5, 0.5 - 1e-12)):
        with pytest.raises(dense.DenseCudaValidationError, match="retention bounds"):
            dense.gated_recurrence(x, minimum_retention=low, maximum_retention=high)
    with pytest.raises(think.CudaThinkValidationError, match="kl_weight finite"):
        think.policy_loss(torch.zeros(4, 9, device=cuda), rows.long(), rows, rows, reference_log_probs=rows, kl_weight=1e39)
