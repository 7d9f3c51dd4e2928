"""Refusals of the training operators: typed errors before any launch, and the C entries' argument checks."""
from __future__ import annotations

import ctypes

import pytest
import torch

from koemi_5hom_b200 import _native
from koemi_5hom_b200.cuda_kernels import core, dense, moe, think
from koemi_5hom_b200.cuda_kernels.loader import CudaExtensionValidationError

cpu_only = pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-CUDA contract")


def test_recurrence_refusals():
    x = torch.rand(2, 3, 8)
    Bad = dense.DenseCudaValidationError
    for call, message in (
            (lambda: dense.gated_recurrence(x[0]), "shape"),
            (lambda: dense.gated_recurrence(x[..., :7]), "2 \\* features"),
            (lambda: dense.gated_recurrence(x.double()), "unsupported CUDA dtype"),
            (lambda: dense.gated_recurrence(x, torch.rand(2, 5)), "initial must be float32"),
            (lambda: dense.gated_recurrence(x, torch.rand(2, 4).bfloat16()), "initial must be float32"),
            (lambda: dense.gated_recurrence(x, valid=torch.ones(2, 4, dtype=torch.bool)), "valid must be bool"),
            (lambda: dense.gated_recurrence(x, restart=torch.ones(2, 3)), "restart must be bool"),
            (lambda: dense.gated_recurrence(x, minimum_retention=0.0), "retention bounds"),
            (lambda: dense.gated_recurrence(x, minimum_retention=0.6, maximum_retention=0.5), "retention bounds"),
            (lambda: dense.gated_recurrence(x, maximum_retention=1.0), "retention bounds"),
            (lambda: dense.gated_recurrence(x, maximum_retention=float("nan")), "retention bounds")):
        with pytest.raises(Bad, match=message):
            call()
    with pytest.raises(TypeError):
        dense.gated_recurrence([1.0])


@cpu_only
def test_recurrence_and_policy_report_unavailable_without_cuda():
    with pytest.raises(dense.DenseCudaUnavailableError):
        dense.gated_recurrence(torch.rand(2, 3, 8))
    with pytest.raises(think.CudaThinkUnavailableError):
        think.policy_loss(torch.rand(4, 9), torch.zeros(4, dtype=torch.long), torch.zeros(4), torch.zeros(4))


def test_route_refusals():
    x = torch.rand(4, 8)
    Bad = moe.CudaMoeValidationError
    for call, message in (
            (lambda: moe.route_learned_topk(x[0], top_k=1), "shape"),
            (lambda: moe.route_learned_topk(x.double(), top_k=1), "float32, float16, or bfloat16"),
            (lambda: moe.route_learned_topk(x, top_k=0), "top_k"),
            (lambda: moe.route_learned_topk(x, top_k=9), "top_k"),
            (lambda: moe.route_learned_topk(x, top_k=True), "top_k"),
            (lambda: moe.route_learned_topk(torch.rand(2, 4097), top_k=1), "limit of 4096"),
            (lambda: moe.route_learned_topk(x, torch.ones(3, dtype=torch.bool), top_k=1), "valid_mask"),
            (lambda: moe.route_learned_topk(x, torch.ones(4), top_k=1), "valid_mask"),
            (lambda: moe.route_learned_topk(x, top_k=1), "must be CUDA tensors")):
        with pytest.raises(Bad, match=message):
            call()
    with pytest.raises(TypeError):
        moe.route_learned_topk([1.0], top_k=1)


def test_policy_refusals():
    logits, t, f = torch.rand(4, 9), torch.zeros(4, dtype=torch.long), torch.zeros(4)
    Bad = think.CudaThinkValidationError
    for call, message in (
            (lambda: think.policy_loss(logits[0], t, f, f), "logits must have shape"),
            (lambda: think.policy_loss(logits.double(), t, f, f), "logits dtype"),
            (lambda: think.policy_loss(logits, t.int(), f, f), "target_ids must be torch.int64"),
            (lambda: think.policy_loss(logits, t, f[:3], f), "old_log_probs"),
            (lambda: think.policy_loss(logits, t, f, f.bfloat16()), "advantages"),
            (lambda: think.policy_loss(logits, t, f, f, valid_mask=f), "valid_mask"),
            (lambda: think.policy_loss(logits, t, f, f, clip_low=-0.1), "clip widths"),
            (lambda: think.policy_loss(logits, t, f, f, clip_high=float("nan")), "clip widths"),
            (lambda: think.policy_loss(logits, t, f, f, kl_weight=0.1), "needs reference_log_probs"),
            (lambda: think.policy_loss(logits, t, f, [0.0]), "must be a torch.Tensor")):
        with pytest.raises(Bad, match=message):
            call()


def test_clip_refusals():
    g = [torch.rand(3)]
    Bad = CudaExtensionValidationError
    for call, message in (
            (lambda: core.clip_gradients(g, -1.0), "max_norm"),
            (lambda: core.clip_gradients(g, float("nan")), "max_norm"),
            (lambda: core.clip_gradients(g, True), "max_norm"),
            (lambda: core.clip_gradients([], 1.0), "must not be empty"),
            (lambda: core.clip_gradients([torch.rand(3).double()], 1.0), "float32, float16 or bfloat16"),
            (lambda: core.clip_gradients([torch.rand(4, 4)[:, 1]], 1.0), "contiguous"),
            (lambda: core.clip_gradients(g, 1.0), "one CUDA device"),
            (lambda: core.gradient_norm(g), "one CUDA device")):
        with pytest.raises(Bad, match=message):
            call()
    with pytest.raises(TypeError):
        core.clip_gradients([[1.0]], 1.0)


@pytest.mark.gpu
def test_refusals_of_cuda_arguments(cuda):
    g = torch.rand(8, device=cuda)
    for out in ([], [g[:4]], [g.bfloat16()], [g.cpu()], [torch.rand(4, 4, device=cuda)[:, :2]]):
        with pytest.raises(CudaExtensionValidationError):
            core.clip_gradients([g], 1.0, out=out)
    with pytest.raises(CudaExtensionValidationError, match="one CUDA device"):
        core.clip_gradients([g, torch.rand(3)], 1.0)
    with pytest.raises(dense.DenseCudaValidationError, match="one CUDA device"):
        dense.gated_recurrence(torch.rand(2, 3, 8, device=cuda), torch.rand(2, 4))
    with pytest.raises(moe.CudaMoeValidationError, match="one device"):
        moe.route_learned_topk(torch.rand(4, 8, device=cuda), torch.ones(4, dtype=torch.bool), top_k=1)
    with pytest.raises(think.CudaThinkValidationError, match="one CUDA device"):
        think.policy_loss(torch.rand(4, 9, device=cuda), torch.zeros(4, dtype=torch.long), torch.zeros(4), torch.zeros(4))


def test_entries_refuse_bad_arguments_before_touching_the_device():
    lib = _native.library()
    invalid, workspace = _native.KOEMI_ERR_INVALID, _native.KOEMI_ERR_WORKSPACE

    def recurrence(batch=1, length=4, features=8, low=0.1, high=0.9, dtype=_native.F32):
        return lib.koemi_dense_gated_recurrence_forward(None, None, None, None, None, None, None, batch, length, features,
                                                        low, high, dtype, None)

    assert recurrence(batch=-1) == invalid and "non-negative" in _native.last_error()
    assert recurrence(low=0.9, high=0.1) == invalid and "retention" in _native.last_error()
    assert recurrence(length=1 << 40) == invalid and "too large" in _native.last_error()
    assert recurrence() == invalid and "non-NULL" in _native.last_error()
    assert recurrence(batch=0) == 0 and recurrence(length=0) == 0 and recurrence(features=0) == 0
    one = ctypes.c_void_p(16)
    assert lib.koemi_dense_gated_recurrence_forward(one, None, None, None, one, one, None, 1, 4, 8, 0.1, 0.9, 99, None) == invalid
    assert lib.koemi_dense_gated_recurrence_backward(None, None, None, None, None, None, None, None, 1, 4, 8, 0.1, 0.9,
                                                     _native.F32, None) == invalid

    size = lib.koemi_moe_route_learned_workspace(100, 8)
    assert size > 0 and lib.koemi_moe_route_learned_workspace(-1, 8) == 0

    def route(tokens=4, experts=8, top_k=2, dtype=_native.F32, room=size):
        return lib.koemi_moe_route_learned_forward(one, None, one, one, one, one, one, tokens, experts, top_k, 0, dtype, one,
                                                   room, None)

    assert route(experts=0) == invalid and route(top_k=9) == invalid and route(tokens=-1) == invalid
    assert route(dtype=99) == invalid and route(room=0) == workspace
    assert lib.koemi_moe_route_learned_backward(None, None, None, None, None, None, None, 4, 8, 2, 0, _native.F32, None) == invalid
    assert lib.koemi_moe_route_learned_backward(None, None, None, None, None, None, None, 0, 8, 2, 0, _native.F32, None) == 0

    def policy(rows=4, vocab=9, inner=4, low=0.2, dtype=_native.F32, room=1 << 20, logits=one):
        return lib.koemi_think_policy_loss_forward(logits, rows, vocab, inner, 0, vocab, one, one, one, None, None, low, 0.2,
                                                   0.0, one, one, one, one, one, None, dtype, one, room, None)

    assert policy(rows=-1) == invalid and policy(vocab=0) == invalid and policy(inner=0) == invalid
    assert policy(low=-1.0) == invalid and policy(logits=None) == invalid and policy(dtype=99) == invalid
    assert policy(room=8) == workspace
    assert lib.koemi_think_policy_loss_backward(None, 4, 9, 4, 0, 9, None, None, None, None, None, None, _native.F32, None) == invalid
    assert lib.koemi_think_policy_loss_scale(None, 4, None, _native.F32, None) == invalid
    assert lib.koemi_think_policy_loss_scale(None, 0, None, _native.F32, None) == 0

    address, elements = (ctypes.c_uint64 * 1)(16), (ctypes.c_int64 * 1)(5)
    code = (ctypes.c_int32 * 1)(_native.F64)

    def clip(count=1, max_norm=1.0, norm=one, room=1 << 20):
        return lib.koemi_core_clip_gradients(address, address, elements, code, count, max_norm, norm, one, room, None)

    assert clip(count=-1) == invalid and clip(max_norm=-1.0) == invalid and clip(norm=None) == invalid
    assert clip() == invalid and "dtype" in _native.last_error()
    code[0], elements[0] = _native.F32, -5
    assert clip() == invalid and "size" in _native.last_error()
    elements[0] = 5
    assert clip(room=0) == workspace
    address[0] = 0
    assert clip() == invalid and "no data" in _native.last_error()
    assert lib.koemi_core_clip_gradients_workspace(elements, 1) >= 4


def test_binding_formats_its_refusals():
    """Its messages are formatted with the process's C++ library, not with one of its own."""
    with pytest.raises(ValueError, match="gradients must be on one CUDA device"):
        _native.binding().koemi_torch_clip_gradients([torch.zeros(2)], None, 1.0)
