"""The training operators called as training programs call them: recomputed, captured, from several threads."""
from __future__ import annotations

import threading

import pytest
import torch
from torch.autograd import forward_ad
from torch.utils.checkpoint import checkpoint

from koemi_5hom_b200.cuda_kernels.core import clip_gradients
from koemi_5hom_b200.cuda_kernels.dense import gated_recurrence
from koemi_5hom_b200.cuda_kernels.moe import route_learned_topk
from koemi_5hom_b200.cuda_kernels.think import policy_loss

pytestmark = pytest.mark.gpu


def recurrence_value(x):
    states, final = gated_recurrence(x)
    return states.float().square().sum() + final.sum()


def route_value(x):
    route = route_learned_topk(x, top_k=2, renormalize=True)
    return route.weights.square().sum() + route.balance_loss


def policy_value(x):
    rows = torch.arange(x.shape[0], device=x.device)
    return policy_loss(x, rows, torch.full_like(rows, -8, dtype=torch.float32), 1.0 + rows.float().cos()).loss / 3


# the scalar of an operator's differentiable outputs, and an input
VALUES = {"recurrence": (recurrence_value, (3, 300, 128), torch.bfloat16), "recurrence step": (recurrence_value, (64, 1, 128), torch.float32),
          "route": (route_value, (300, 64), torch.float32), "policy": (policy_value, (30, 5000), torch.bfloat16),
          "policy of short rows": (policy_value, (30, 257), torch.float32), "policy of long rows": (policy_value, (30, 70000), torch.float16)}


@pytest.fixture(params=VALUES, ids=VALUES)
def operator(request, cuda):
    value, shape, dtype = VALUES[request.param]
    return value, torch.randn(shape, generator=torch.Generator().manual_seed(1)).to(dtype).to(cuda)


def test_activation_checkpointing_gives_the_same_bits(operator):
    value, x = operator
    grads = []
    for run in (value, lambda t: checkpoint(value, t, use_reentrant=False)):
        leaf = x.clone().requires_grad_(True)
        grads.append(torch.autograd.grad(run(leaf), leaf)[0])
    assert torch.equal(*grads) and grads[0].any()


def test_forward_mode_is_refused(operator, cuda):
    value, x = operator
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        value(forward_ad.make_dual(x, torch.ones_like(x)))
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        clip_gradients([forward_ad.make_dual(x, torch.ones_like(x))], 1.0)


def test_functional_gradients_give_the_same_bits(operator):
    value, x = operator
    leaf = x.clone().requires_grad_(True)
    want, = torch.autograd.grad(value(leaf), leaf)
    assert torch.equal(torch.func.grad(value)(x), want)


# calls of one kernel with different needs of shared memory
SIZES = {"policy": (policy_value, [(4, v) for v in (32768, 20000, 17000, 30000)], torch.bfloat16),
         "recurrence": (recurrence_value, [(1, 2100, 64), (40, 300, 512), (1, 600, 64)], torch.bfloat16),
         "route": (route_value, [(5, e) for e in (4096, 300, 2000)], torch.float32)}


@pytest.mark.parametrize("name", SIZES)
def test_threads_with_different_sizes(name, cuda):
    """One thread's call never takes from another's launch the shared memory that it needs."""
    value, shapes, dtype = SIZES[name]
    errors = []

    def work(shape):
        try:
            x = torch.randn(shape, device=cuda).to(dtype)
            with torch.no_grad():
                for _ in range(1500):
                    value(x)
        except Exception as error:  # noqa: BLE001
            errors.append(error)

    threads = [threading.Thread(target=work, args=(shape,)) for shape in shapes]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not errors, errors[0]


@pytest.mark.parametrize("value,shape,dtype", [(recurrence_value, (1, 9000, 64), torch.bfloat16), (recurrence_value, (2, 5000, 96), torch.float32),
                                               (policy_value, (600, 70000), torch.bfloat16), (policy_value, (40, 131072), torch.float32)])
def test_exchanges_inside_clusters_repeat(value, shape, dtype, cuda):
    """Long chains and long rows, whose parts CTAs of a cluster store into each other's memory, give equal bits each time."""
    x = torch.randn(shape, generator=torch.Generator().manual_seed(5)).to(dtype).to(cuda).requires_grad_(True)
    results = []
    for _ in range(12):
        result = value(x)
        results.append((result.detach(), *torch.autograd.grad(result, x)))
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))


def test_forward_and_backward_in_a_cuda_graph(operator):
    value, x = operator
    x.requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            torch.autograd.grad(value(x), x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        result = value(x)
        grad, = torch.autograd.grad(result, x)
    with torch.no_grad():
        x.copy_(x.flip(0))
    graph.replay()
    expected = value(x)
    assert torch.equal(result, expected) and torch.equal(grad, torch.autograd.grad(expected, x)[0])
