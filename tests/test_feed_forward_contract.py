"""Refusals of the feed-forward sub-layer's operators, their C entries' argument checks, and what torch records of them."""
from __future__ import annotations

import ctypes

import pytest
import torch
from torch.autograd import forward_ad
from torch.utils.checkpoint import checkpoint

from koemi_5hom_b200 import _native
from koemi_5hom_b200.cuda_kernels import _training, core, dense
from koemi_5hom_b200.cuda_kernels.loader import CudaExtensionUnavailableError, CudaExtensionValidationError

cpu_only = pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-CUDA contract")


def refused(calls, error):
    for call, message in calls:
        with pytest.raises(error, match=message):
            call()


def test_layer_norm_refusals():
    x, w = torch.rand(2, 3, 8), torch.rand(8)
    refused(((lambda: core.layer_norm(torch.tensor(1.0), w), "shape"),
             (lambda: core.layer_norm(torch.rand(3, 0), torch.rand(0)), "positive width"),
             (lambda: core.layer_norm(x.double(), w), "found torch.float64"),
             (lambda: core.layer_norm(x, torch.rand(7)), "weight must have shape"),
             (lambda: core.layer_norm(x, w, torch.rand(1, 8)), "bias must have shape"),
             (lambda: core.layer_norm(x, w.bfloat16()), "weight must use torch.float32"),
             (lambda: core.layer_norm(x.bfloat16(), w.half()), "weight must use torch.bfloat16 or float32"),
             (lambda: core.layer_norm(x.bfloat16(), w, w.bfloat16()), "same dtype"),
             (lambda: core.layer_norm(x, w, eps=-1.0), "eps"),
             (lambda: core.layer_norm(x, w, eps=float("nan")), "eps"),
             (lambda: core.layer_norm(x, w, eps=float("inf")), "eps"),
             (lambda: core.layer_norm(x, w, eps=True), "eps")), CudaExtensionValidationError)
    for call in (lambda: core.layer_norm([1.0], w), lambda: core.layer_norm(x, None), lambda: core.layer_norm(x, w, 0.5)):
        with pytest.raises(TypeError):
            call()


def test_dropout_refusals():
    x = torch.rand(2, 3)
    refused(((lambda: core.dropout(x, -0.1, seed=1), "probability"),
             (lambda: core.dropout(x, 1.5, seed=1), "probability"),
             (lambda: core.dropout(x, float("nan"), seed=1), "probability"),
             (lambda: core.dropout(x, True, seed=1), "probability"),
             (lambda: core.dropout(x, 0.1, seed=-1), "seed"),
             (lambda: core.dropout(x, 0.1, seed=1 << 64), "seed"),
             (lambda: core.dropout(x, 0.1, seed=1.0), "seed"),
             (lambda: core.dropout(x, 0.1, seed=1, site=-2), "site"),
             (lambda: core.dropout(x, 0.1, seed=1, step=None), "step"),
             (lambda: core.dropout(x, 0.1, seed=1, step=torch.zeros(1, dtype=torch.int64)), "zero-dimensional int64"),
             (lambda: core.dropout(x, 0.1, seed=1, step=torch.tensor(1.0)), "zero-dimensional int64"),
             (lambda: core.dropout(x.double(), 0.1, seed=1), "float64"),
             (lambda: core.dropout(x, 0.1, seed=1, residual=torch.rand(3, 2)), "residual"),
             (lambda: core.dropout(x, 0.1, seed=1, residual=x.half()), "residual")), CudaExtensionValidationError)
    for call in (lambda: core.dropout([1.0], 0.1, seed=1), lambda: core.dropout(x, 0.1, seed=1, residual=1.0)):
        with pytest.raises(TypeError):
            call()


def test_block_refusals():
    x, g, v, o = torch.rand(2, 3, 8), torch.rand(16, 8), torch.rand(16, 8), torch.rand(4, 16)
    block = dense.gated_feed_forward
    refused(((lambda: block(torch.tensor(1.0), g, v, o), "shape"),
             (lambda: block(torch.rand(2, 0), torch.rand(4, 0), torch.rand(4, 0), torch.rand(2, 4)), "positive width"),
             (lambda: block(x.double(), g, v, o), "unsupported CUDA dtype"),
             (lambda: block(x, g[0], v, o), "gate_weight must have shape"),
             (lambda: block(x, g[:, :7], v[:, :7], o), "gate_weight must have shape"),
             (lambda: block(x, g[:0], v[:0], o[:, :0]), "gate_weight must have shape"),
             (lambda: block(x, g, v[:15], o), "value_weight must have shape"),
             (lambda: block(x, g, v, o[:, :15]), "output_weight must have shape"),
             (lambda: block(x, g, v, o[:0]), "output_weight must have shape"),
             (lambda: block(x, g, v, o, gate_bias=torch.rand(15)), "gate_bias must have shape"),
             (lambda: block(x, g, v, o, output_bias=torch.rand(1, 4)), "output_bias must have shape"),
             (lambda: block(x, g, v.half(), o), "value_weight must use"),
             (lambda: block(x.half(), g.half(), v.half(), o.half(), value_bias=torch.rand(16)), "value_bias must use")),
            dense.DenseCudaValidationError)
    for call in (lambda: block([1.0], g, v, o), lambda: block(x, None, v, o), lambda: block(x, g, v, o, value_bias=1.0)):
        with pytest.raises(TypeError):
            call()


@cpu_only
def test_block_reports_unavailable_without_cuda():
    with pytest.raises(dense.DenseCudaUnavailableError):
        dense.gated_feed_forward(torch.rand(2, 8), torch.rand(16, 8), torch.rand(16, 8), torch.rand(4, 16))


@cpu_only
def test_cpu_tensors_are_refused():
    x, w = torch.rand(2, 8), torch.rand(8)
    for call in (lambda: core.layer_norm(x, w), lambda: core.dropout(x, 0.1, seed=1)):
        with pytest.raises((CudaExtensionValidationError, CudaExtensionUnavailableError)):
            call()


@pytest.mark.gpu
def test_tensors_of_another_device_are_refused(cuda):
    x, w = torch.rand(2, 8, device=cuda), torch.rand(8, device=cuda)
    refused(((lambda: core.layer_norm(x, w.cpu()), "one CUDA device"), (lambda: core.layer_norm(x.cpu(), w), "one CUDA device"),
             (lambda: core.layer_norm(x, w, w.cpu()), "one CUDA device"), (lambda: core.dropout(x.cpu(), 0.1, seed=1), "one CUDA device"),
             (lambda: core.dropout(x, 0.1, seed=1, residual=x.cpu()), "one CUDA device"),
             (lambda: core.dropout(x, 0.1, seed=1, step=torch.tensor(1)), "one CUDA device")), CudaExtensionValidationError)
    g, o = torch.rand(16, 8, device=cuda), torch.rand(4, 16, device=cuda)
    refused(((lambda: dense.gated_feed_forward(x, g, g.cpu(), o), "one CUDA device"),
             (lambda: dense.gated_feed_forward(x.cpu(), g, g, o), "one CUDA device"),
             (lambda: dense.gated_feed_forward(x, g, g, o, output_bias=torch.rand(4)), "one CUDA device")), dense.DenseCudaValidationError)


def test_entries_refuse_bad_arguments_before_touching_the_device():
    lib = _native.library()
    invalid, workspace = _native.KOEMI_ERR_INVALID, _native.KOEMI_ERR_WORKSPACE
    one = ctypes.c_void_p(16)

    def norm(rows=4, width=8, inner=4, stride=8, weight=one, weight_dtype=_native.F32, eps=1e-5, dtype=_native.F32, values=one):
        return lib.koemi_core_layer_norm_forward(values, rows, width, inner, 0, stride, weight, None, weight_dtype, one, None, eps, dtype, None)

    assert norm(rows=-1) == invalid and norm(width=0) == invalid and norm(inner=0) == invalid and norm(stride=-8) == invalid
    assert norm(rows=1 << 40) == invalid and norm(width=1 << 40) == invalid
    assert norm(dtype=99) == invalid and norm(weight_dtype=_native.BF16) == invalid and norm(eps=-1.0) == invalid
    assert norm(eps=float("nan")) == invalid and norm(eps=float("inf")) == invalid and norm(values=None) == invalid
    assert norm(weight=None) == invalid and norm(values=ctypes.c_void_p(17)) == invalid
    assert norm(rows=0) == 0

    size = lib.koemi_core_layer_norm_backward_workspace(4, 8)
    assert size == 4 * 2 * 8 * 4 and lib.koemi_core_layer_norm_backward_workspace(-1, 8) == 0
    assert lib.koemi_core_layer_norm_backward_workspace(1 << 30, 8) == 1024 * 2 * 8 * 4

    def norm_backward(rows=4, dtype=_native.F32, stats=one, room=size):
        return lib.koemi_core_layer_norm_backward(one, rows, 8, 4, 0, 8, one, _native.F32, stats, one, one, one, one, dtype, one, room, None)

    assert norm_backward(rows=-1) == invalid and norm_backward(dtype=_native.I64) == invalid and norm_backward(stats=None) == invalid
    assert norm_backward(room=size - 1) == workspace

    def drop(count=4, dropped=100, dtype=_native.F32, values=one):
        return lib.koemi_core_dropout(values, None, one, count, dropped, 1, 2, 3, None, dtype, None)

    kept = lib.koemi_dense_gated_feed_forward_kept(10, 20, _native.BF16)
    assert kept == 768 + 2 * 4096 and lib.koemi_dense_gated_feed_forward_kept(-1, 20, _native.BF16) == 0  # 10 x 32 values, twice 32 x 32 in fp32
    assert lib.koemi_dense_gated_feed_forward_kept(10, 20, _native.F32) == 2048 + 2 * 4096  # three bf16 parts
    rooms = [lib.koemi_dense_gated_feed_forward_workspace(10, 16, 20, 8, _native.BF16, backward) for backward in (0, 1)]
    assert min(rooms) > 0 and lib.koemi_dense_gated_feed_forward_workspace(10, 16, 20, 8, 99, 0) == 0
    page = ctypes.c_void_p(256)

    def block(rows=10, width=16, hidden=20, out=8, stride=16, dtype=_native.BF16, values=page, keep=page, keep_bytes=kept, room=rooms[0], ws=page):
        return lib.koemi_dense_gated_feed_forward_forward(values, stride, page, page, page, None, None, None, page, keep, keep_bytes, rows,
                                                          width, hidden, out, dtype, ws, room, None)

    assert block(rows=-1) == invalid and block(width=0) == invalid and block(hidden=0) == invalid and block(out=0) == invalid
    assert block(rows=1 << 31) == invalid and block(hidden=1 << 25) == invalid and block(stride=15) == invalid
    assert block(dtype=_native.I32) == invalid and block(values=None) == invalid and block(rows=0) == 0
    assert block(keep_bytes=kept - 1) == workspace and block(keep=one) == workspace
    assert block(room=8) == workspace and block(ws=None) == workspace and block(ws=one) == workspace

    def block_backward(rows=10, stride=16, dtype=_native.BF16, keep=page, grad=page, room=rooms[1]):
        return lib.koemi_dense_gated_feed_forward_backward(page, stride, page, page, page, keep, kept, grad, page, page, page, page, page, page,
                                                           page, rows, 16, 20, 8, dtype, page, room, None)

    assert block_backward(rows=-1) == invalid and block_backward(stride=3) == invalid and block_backward(dtype=99) == invalid
    assert block_backward(keep=None) == invalid and block_backward(grad=None) == invalid and block_backward(keep=one) == workspace
    assert block_backward(room=8) == workspace

    assert drop(count=-1) == invalid and drop(dropped=-1) == invalid and drop(dropped=65537) == invalid
    assert drop(dtype=_native.BOOL) == invalid and drop(values=None) == invalid and drop(count=0) == 0


# ------------------------------------- in torch's own machinery, on meta tensors

def norm_value(x):
    return torch.ops.koemi_b200.layer_norm(x, x[0].detach() + 1, x[0], 1e-5).sum()


def dropout_value(x):
    return torch.ops.koemi_b200.dropout(x, 2 * x, None, 6554, 1, 2, 3).sum()


def block_value(x):
    return torch.ops.koemi_b200.gated_feed_forward(x.view(2, 3, 16), x[0].expand(8, 16), x[1:2].expand(8, 16), x[:4, :8], x[0, :8], None, x[1, :4]).sum()


SCALARS = {"norm": norm_value, "dropout": dropout_value, "block": block_value}


@pytest.fixture(params=SCALARS, ids=SCALARS)
def operator(request):
    _training.register()
    return SCALARS[request.param], torch.zeros(6, 16, device="meta")


def test_activation_checkpointing_and_functional_gradients(operator):
    value, x = operator
    leaf = x.clone().requires_grad_(True)
    grad, = torch.autograd.grad(checkpoint(lambda t: value(2 * t), leaf, use_reentrant=False), leaf)
    assert grad.shape == x.shape and torch.func.grad(value)(x).shape == x.shape


def test_forward_mode_is_refused(operator):
    value, x = operator
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        value(forward_ad.make_dual(x, torch.ones_like(x)))


@pytest.mark.parametrize("value", [norm_value, block_value])
def test_second_orders_are_refused(value):
    _training.register()
    x = torch.zeros(6, 16, device="meta")
    with pytest.raises(RuntimeError, match="not implemented"):
        torch.func.grad(lambda t: torch.func.grad(value)(t).sum())(x)
    leaf = x.requires_grad_(True)
    with pytest.raises(RuntimeError, match="first order"):
        torch.autograd.grad(value(leaf), leaf, create_graph=True)


def test_dropout_has_every_order():
    _training.register()
    x = torch.zeros(6, 16, device="meta", requires_grad=True)
    grad, = torch.autograd.grad((dropout_value(x) ** 2).sum(), x, create_graph=True)
    assert torch.autograd.grad(grad.sum(), x)[0].shape == x.shape
    assert torch.func.grad(lambda t: torch.func.grad(dropout_value)(t).sum() + t.sum())(x.detach()).shape == x.shape
