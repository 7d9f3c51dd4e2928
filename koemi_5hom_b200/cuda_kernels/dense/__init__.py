from koemi_5hom_b200.cuda_kernels.dense.affine_scan import (
    DenseCudaBuildError,
    DenseCudaUnavailableError,
    DenseCudaValidationError,
    dense_affine_scan,
    native_cuda_available,
)
from koemi_5hom_b200.cuda_kernels.dense.feed_forward import gated_feed_forward
from koemi_5hom_b200.cuda_kernels.dense.gated_recurrence import gated_recurrence

__all__ = [
    "DenseCudaBuildError",
    "DenseCudaUnavailableError",
    "DenseCudaValidationError",
    "dense_affine_scan",
    "gated_feed_forward",
    "gated_recurrence",
    "native_cuda_available",
]
