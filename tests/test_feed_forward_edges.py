"""Corners of the feed-forward sub-layer's operators that need no GPU: what their C entries and torch's transforms are
refused, what they ask for, and the arithmetic of fp32 values in bf16 parts."""
from __future__ import annotations

import ctypes

import pytest
import torch

from koemi_5hom_b200 import _native
from koemi_5hom_b200.cuda_kernels import _training

PAGE = 256  # an address that nothing reads


def pointers(names, odd, by):
    """PAGE for every name, `by` bytes behind it for `odd`."""
    return {name: ctypes.c_void_p(PAGE + (by if name == odd else 0)) for name in names}


@pytest.mark.parametrize("dtype", [_native.F32, _native.BF16])
def test_entries_refuse_pointers_off_their_type(dtype):
    """Before anything is launched: on the device such an access would end the context."""
    lib, invalid = _native.library(), _native.KOEMI_ERR_INVALID
    half = 2 if dtype == _native.F32 else 1
    names = ("values", "weight", "bias", "out", "stats")
    for odd in names:
        p = pointers(names, odd, 2 if odd == "stats" else half)
        assert lib.koemi_core_layer_norm_forward(p["values"], 4, 8, 4, 0, 8, p["weight"], p["bias"], dtype, p["out"], p["stats"], 1e-5, dtype,
                                                 None) == invalid, odd
    names = ("values", "weight", "stats", "grad", "dx", "dw", "db", "workspace")
    for odd in names:
        p = pointers(names, odd, {"stats": 2, "workspace": 8}.get(odd, half))
        assert lib.koemi_core_layer_norm_backward(p["values"], 4, 8, 4, 0, 8, p["weight"], dtype, p["stats"], p["grad"], p["dx"], p["dw"], p["db"],
                                                  dtype, p["workspace"], 1 << 20, None) == (_native.KOEMI_ERR_WORKSPACE if odd == "workspace" else invalid), odd
    names = ("values", "residual", "out", "step")
    for odd in names:
        p = pointers(names, odd, 4 if odd == "step" else half)
        assert lib.koemi_core_dropout(p["values"], p["residual"], p["out"], 9, 100, 1, 2, 3, p["step"], dtype, None) == invalid, odd
    names = ("values", "wg", "wv", "wo", "bg", "bv", "bo", "out")
    for odd in names:
        p = pointers(names, odd, half)
        assert lib.koemi_dense_gated_feed_forward_forward(p["values"], 16, *(p[n] for n in names[1:]), None, 0, 10, 16, 20, 8, dtype,
                                                          ctypes.c_void_p(PAGE), 1 << 24, None) == invalid, odd
    names = ("values", "wg", "wv", "wo", "grad", "dx", "dwg", "dwv", "dwo", "dbg", "dbv", "dbo")
    for odd in names:
        p = pointers(names, odd, half)
        assert lib.koemi_dense_gated_feed_forward_backward(p["values"], 16, p["wg"], p["wv"], p["wo"], ctypes.c_void_p(PAGE), 1 << 20,
                                                           *(p[n] for n in names[4:]), 10, 16, 20, 8, dtype, ctypes.c_void_p(PAGE), 1 << 24,
                                                           None) == invalid, odd


@pytest.mark.parametrize("batched", ["values", "residual"])
def test_dropout_is_refused_under_vmap(batched):
    """Called once a sample it would name the same positions' bits, the same mask, for every one of them."""
    _training.register()
    x, r = torch.zeros(5, 6, 16, device="meta"), torch.zeros(6, 16, device="meta")
    drop = lambda t: torch.ops.koemi_b200.dropout(*((t, r) if batched == "values" else (r, t)), None, 6554, 1, 2, 3)  # noqa: E731
    assert drop(x[0]).shape == r.shape
    for call in (drop, torch.func.grad(lambda t: drop(t).sum())):
        with pytest.raises(NotImplementedError, match="vmap"):
            torch.vmap(call)(x)


def test_block_workspace_is_what_the_pass_uses():
    """Bits of the query's last argument: 1 the backward, 2 the forward writes kept, 4 every operand starts at a
    multiple of 16 bytes with rows of a multiple of 8 values. 0 and 1 ask for enough for any operands."""
    ask = _native.library().koemi_dense_gated_feed_forward_workspace
    sizes, rows, hidden = (32768, 2048, 4096, 2048), 32768, 4096
    operands = 2 * (rows * 2048 + 3 * 4096 * 2048)  # x and the weights in padded rows
    assert ask(*sizes, _native.BF16, 0) >= 2 * rows * hidden + operands
    assert 2 * rows * hidden <= ask(*sizes, _native.BF16, 4) < 2 * rows * hidden + 2 ** 20  # h
    assert 0 < ask(*sizes, _native.BF16, 2 | 4) < 2 ** 20
    assert operands <= ask(*sizes, _native.BF16, 2) < operands + 2 ** 20
    both = 4 * rows * hidden  # dp and dq
    assert both <= ask(*sizes, _native.BF16, 1 | 4) < both + 2 ** 21 and ask(*sizes, _native.BF16, 1) >= both + operands + 2 * rows * 2048
    for dtype in (_native.F32, _native.BF16):  # fp32 operands are always split, odd rows always copied
        for odd in ((300, 515, 1030, 515), (3, 515, 77, 33)):
            assert ask(*odd, dtype, 0) == ask(*odd, dtype, 4) and ask(*odd, dtype, 1) == ask(*odd, dtype, 1 | 4)
            assert 0 < ask(*odd, dtype, 2) <= ask(*odd, dtype, 0)


def test_norm_workspace_holds_the_partial_rows_that_there_are():
    """A wide row takes many threads, so an SM holds few CTAs, each with one partial row of dw and db: 8 an SM of 2048
    columns, 1 an SM from 16384 on; never more than rows."""
    ask = _native.library().koemi_core_layer_norm_backward_workspace
    for width in (1, 128, 2000):
        assert ask(1 << 20, width) == 1024 * 2 * width * 4
    sms = ask(1 << 20, 1 << 20) // (2 * 4 << 20)
    assert 1 <= sms <= 512
    for width, each in ((4096, 4), (5000, 3), (8192, 2), (12000, 1), (16384, 1), (33000, 1)):
        assert ask(1 << 20, width) == min(1024, each * sms) * 2 * width * 4
        assert ask(7, width) == 7 * 2 * width * 4


def test_three_bf16_parts_hold_an_fp32_value():
    """Every fp32 value of a binade: the parts add up to it exactly, and the products of parts that the block leaves out,
    x1 y2, x2 y1 and x2 y2, are one fp32 rounding of x y at most (the parts' bounds make it 2^-24 + 2^-34 of x0 y0)."""
    x = torch.arange(1 << 23, dtype=torch.int32).add_(0x3F800000).view(torch.float32)
    parts, rest = [], x
    for _ in range(3):
        parts.append(rest.bfloat16().float())
        rest = rest - parts[-1]
    assert not rest.any()
    x0, x1, x2 = (t.double() for t in parts)
    assert (x1 / x0).abs().max().item() == 2.0 ** -8 and (x2 / x0).abs().max().item() <= 2.0 ** -17
    for order in (torch.arange(1 << 23), torch.randperm(1 << 23, generator=torch.Generator().manual_seed(0))):
        y0, y1, y2 = x0[order], x1[order], x2[order]
        left_out = ((x1 * y2 + x2 * y1 + x2 * y2) / (x.double() * x.double()[order])).abs().max().item()
        assert left_out <= 1.01 * 2.0 ** -24


def test_dropout_has_batched_gradients():
    """Rows of a Jacobian share the forward's mask: there vmap calls the gradient's operator, not dropout."""
    _training.register()
    x = torch.zeros(6, 16, device="meta", requires_grad=True)
    drop = lambda t: torch.ops.koemi_b200.dropout(t, 2 * t, None, 6554, 1, 2, 3)  # noqa: E731
    grad, = torch.autograd.grad(drop(x), x, torch.zeros(5, 6, 16, device="meta"), is_grads_batched=True)
    assert grad.shape == (5, 6, 16)
    assert torch.func.jacrev(drop)(x.detach()).shape == (6, 16, 6, 16)
    assert torch.func.jacrev(torch.func.jacrev(lambda t: drop(t * t).sum()))(x.detach()[:1]).shape == (1, 16, 1, 16)


@pytest.mark.parametrize("call", [lambda x: torch.ops.koemi_b200.layer_norm(x, x[0].detach() + 1, x[0], 1e-5),
                                  lambda x: torch.ops.koemi_b200.gated_feed_forward(x, x[:1].expand(8, 16), x[1:2].expand(8, 16), x[:4, :8], None, None, x[1, :4])])
def test_norm_and_block_have_batched_gradients(call):
    _training.register()
    x = torch.zeros(6, 16, device="meta", requires_grad=True)
    y = call(x)
    grad, = torch.autograd.grad(y, x, torch.zeros(5, *y.shape, device="meta"), is_grads_batched=True)
    assert grad.shape == (5, 6, 16) and torch.func.jacrev(call)(x.detach()).shape == (*y.shape, 6, 16)
