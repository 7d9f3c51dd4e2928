"""The training operators in torch's own machinery, on meta tensors: nothing is computed, everything is recorded."""
from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest
import torch
from torch.autograd import forward_ad
from torch.utils.checkpoint import checkpoint

from koemi_5hom_b200.cuda_kernels import _training

ROOT = Path(__file__).resolve().parent.parent


def test_first_calls_from_several_threads():
    """Both threads come to the registration before either has finished it."""
    code = """
import threading, time
from koemi_5hom_b200 import _native
from koemi_5hom_b200.cuda_kernels import _training
binding, errors = _native.binding, []
def slow():
    time.sleep(0.5)
    return binding()
_native.binding = slow
import torch
_native.ensure_device = lambda device: None
def call():
    try:
        _training.load(torch.device("cuda", 0))
    except Exception as error:
        errors.append(error)
threads = [threading.Thread(target=call) for _ in range(4)]
for t in threads: t.start()
for t in threads: t.join()
assert not errors, errors
assert _training.loaded()
"""
    result = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert result.returncode == 0, result.stderr


def recurrence(x, initial=None):
    return torch.ops.koemi_b200.gated_recurrence(x, initial, None, None, 0.1, 0.9)


def route(logits):
    return torch.ops.koemi_b200.route_learned(logits, None, 2, False)


def policy(logits, old=None, advantages=None, reference=None):
    rows = torch.zeros(6, device="meta")
    targets = torch.zeros(6, dtype=torch.int64, device="meta")
    return torch.ops.koemi_b200.policy_loss(logits, targets, rows if old is None else old, rows if advantages is None else advantages,
                                            reference, None, 0.2, 0.2, 0.0)


# an operator's scalar of its differentiable outputs, and the shape of its input
SCALARS = {"recurrence": (lambda x: sum(t.sum() for t in recurrence(x)), (2, 40, 16)),
           "route": (lambda x: route(x)[1].sum() + route(x)[3], (6, 9)),
           "policy": (lambda x: policy(x)[0], (6, 9))}


@pytest.fixture(params=SCALARS, ids=SCALARS)
def operator(request):
    _training.register()
    value, shape = SCALARS[request.param]
    return value, torch.zeros(shape, device="meta")


@pytest.mark.parametrize("before", [False, True])
def test_activation_checkpointing(operator, before):
    """The recomputation inside the node's unpacking is recorded, as it is for torch's own operators."""
    value, x = operator
    leaf = x.clone().requires_grad_(True)
    out = checkpoint(lambda t: value(2 * t if before else t), leaf, use_reentrant=False)
    grad, = torch.autograd.grad(out, leaf)
    assert grad.shape == x.shape


def test_forward_mode_is_refused(operator):
    """A tangent is never dropped without a word."""
    value, x = operator
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        value(forward_ad.make_dual(x, torch.ones_like(x)))
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(value, (x,), (torch.ones_like(x),))
    with forward_ad.dual_level():  # no tangent of this level: as ever
        value(x)


def test_forward_mode_of_the_other_inputs_is_refused():
    _training.register()
    rows, logits = torch.zeros(6, device="meta"), torch.zeros(6, 9, device="meta")
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(rows, torch.ones_like(rows))
        for call in (lambda: policy(logits, old=dual), lambda: policy(logits, advantages=dual), lambda: policy(logits, reference=dual),
                     lambda: recurrence(torch.zeros(2, 3, 4, device="meta"), forward_ad.make_dual(torch.zeros(2, 2, device="meta"),
                                                                                                  torch.ones(2, 2, device="meta")))):
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                call()


def test_functional_gradients_of_first_order(operator):
    value, x = operator
    assert torch.func.grad(value)(x).shape == x.shape
    grad, result = torch.func.grad_and_value(value)(x)
    assert grad.shape == x.shape and result.shape == ()


def test_second_orders_are_refused(operator):
    """By torch.func inside itself, by autograd around it, and by create_graph."""
    value, x = operator
    first = torch.func.grad(value)
    with pytest.raises(RuntimeError, match="not implemented"):
        torch.func.grad(lambda t: first(t).sum())(x)
    leaf = x.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="not implemented"):
        torch.autograd.grad(first(leaf).sum(), leaf)
    with pytest.raises(RuntimeError, match="first order"):
        torch.autograd.grad(value(leaf), leaf, create_graph=True)
