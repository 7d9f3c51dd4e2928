from koemi_5hom_b200.cuda_kernels.core.clip_gradients import clip_gradients, gradient_norm
from koemi_5hom_b200.cuda_kernels.core.dropout import dropout
from koemi_5hom_b200.cuda_kernels.core.layer_norm import layer_norm
from koemi_5hom_b200.cuda_kernels.core.rmsnorm_silu import (
    fused_rmsnorm_silu,
    gated_rmsnorm_silu,
    load_core_extension,
    rms_norm,
)

__all__ = [
    "clip_gradients",
    "dropout",
    "fused_rmsnorm_silu",
    "gated_rmsnorm_silu",
    "gradient_norm",
    "layer_norm",
    "load_core_extension",
    "rms_norm",
]
