"""Layer norm and dropout on the GPU against plain 64-bit forms (oracle/feed_forward.py).

A result of type T may be off by its own rounding, U[T] relative, plus what the
fp32 arithmetic in front of it loses, counted in roundings (EPS = 2^-24) of the
terms that the formula adds up at that very entry.
"""
from __future__ import annotations

import pytest
import torch

from koemi_5hom_b200.cuda_kernels.core import dropout, layer_norm
from oracle import feed_forward as plain

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}  # fp16: half the subnormal spacing
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def check(got, exact, allowed):
    """|got - exact| <= U |exact| + allowed, elementwise (allowed: a tensor of the results' shape, or a number)."""
    dtype, got, exact = got.dtype, got.detach().double(), exact.detach().double()
    over = (got - exact).abs() - (U[dtype] * 1.0001 * exact.abs() + allowed + TINY[dtype])
    assert got.shape == exact.shape and not got.isnan().any()
    assert not got.numel() or over.max().item() <= 0, f"off by {over.max().item()} more than allowed"


# ---------------------------------------------------------------- layer norm

def norm_with_bounds(x, w, b, g, eps):
    """64-bit (y, dx, dw, db) and what fp32 may lose of each, entry by entry.

    A sum over a row is at most width / 1024 + 40 additions deep (a thread's
    own, two trees of 5, the exchange), so the mean is off by that many EPS of
    mean |x| and the variance by as many EPS of itself; 1 / sqrt, its argument
    and the products are counted as 8 more. A sum over rows is at most rows / 148
    + 100 additions deep: a CTA's own rows, 8 warps, and the partial rows.
    """
    x, w, g = x.double(), w.double(), g.double()
    rows, width = x.shape
    deep, down = (width / 1024 + 40) * EPS, (rows / 148 + 100) * EPS
    mean = x.mean(-1, keepdim=True)
    inverse = ((x - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
    u = (x - mean) * inverse
    u_lost = inverse * (deep * x.abs().mean(-1, keepdim=True) + 2 * EPS * (x - mean).abs()) + u.abs() * (deep + 8 * EPS)
    y = u * w + (0 if b is None else b.double())
    y_lost = w.abs() * u_lost + 2 * EPS * ((u * w).abs() + y.abs())
    a = g * w
    first, second = a.mean(-1, keepdim=True), (a * u).mean(-1, keepdim=True)
    first_lost = 2 * deep * a.abs().mean(-1, keepdim=True)
    second_lost = 2 * deep * (a * u).abs().mean(-1, keepdim=True) + (a.abs() * u_lost).mean(-1, keepdim=True)
    dx = inverse * (a - first - u * second)
    terms = a.abs() + first.abs() + (u * second).abs()
    dx_lost = inverse * (first_lost + u.abs() * second_lost + u_lost * second.abs() + (deep + 12 * EPS) * terms)
    dw, db = (g * u).sum(0), g.sum(0)
    dw_lost = (g.abs() * u_lost).sum(0) + 2 * down * (g * u).abs().sum(0)
    return (y, y_lost), (dx, dx_lost), (dw, dw_lost), (db, 2 * down * g.abs().sum(0))


def norm_case(rows, width, dtype, wide, bias, cuda, seed=0):
    gen = torch.Generator().manual_seed(rows * 7919 + width + seed)
    x = (torch.randn(rows, width, generator=gen) * torch.exp(torch.randn(rows, 1, generator=gen)) + 0.5).to(dtype).to(cuda)
    kind = torch.float32 if wide else dtype
    w = (1 + 0.2 * torch.randn(width, generator=gen)).to(kind).to(cuda)
    b = (0.3 * torch.randn(width, generator=gen)).to(kind).to(cuda) if bias else None
    return x, w, b, torch.randn(rows, width, generator=gen).to(dtype).to(cuda)


def check_norm(x, w, b, g, eps=1e-5):
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b) if t is not None]
    y = layer_norm(*leaves, eps=eps)
    got = (y, *torch.autograd.grad(y, leaves, g))
    with torch.no_grad():
        assert torch.equal(layer_norm(x, w, b, eps=eps), y)
    assert y.dtype == x.dtype and [t.dtype for t in got[1:]] == [t.dtype for t in leaves]
    for t, (exact, lost) in zip(got, norm_with_bounds(x, w, b, g, eps)):
        check(t, exact, lost)


WIDTHS = [1, 2, 7, 8, 33, 64, 128, 255, 512, 515, 520, 1021, 1024, 2048, 4096, 4100, 8192, 8200, 16384, 16400, 33000]


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", WIDTHS)
def test_norm_and_gradients_match_the_plain_form(width, dtype, wide, cuda):
    for rows, bias in ((1, True), (19, width % 2 == 0)):
        check_norm(*norm_case(rows, width, dtype, wide, bias, cuda))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width", [(5000, 64), (20011, 96), (4099, 1021), (3001, 2048), (700, 9000)])
def test_norm_of_many_rows(rows, width, dtype, cuda):
    """More rows than the backward's grid holds at once."""
    check_norm(*norm_case(rows, width, dtype, True, True, cuda))


STRIDED = {"shorter": lambda t: t[:, :-1, :256], "later": lambda t: t[:, 3:, 8:], "one batch, off 16 bytes": lambda t: t[2, :, 1:257],
           "off 16 bytes": lambda t: t[:, :, 5:261], "repeated": lambda t: t[:, 0, :256].unsqueeze(1).expand(6, 9, 256),
           "columns apart": lambda t: t[:, :, 8:].transpose(1, 2), "four dimensions": lambda t: t[..., :256].reshape(2, 3, 40, 256),
           "flat, off 16 bytes": lambda t: t.flatten()[1:1 + 256 * 5].view(5, 256)}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("view", STRIDED)
def test_norm_of_strided_and_offset_rows(view, dtype, cuda):
    """Rows that the vector loads fit and rows that they do not fit add up in different orders, so both are held to the exact form."""
    gen = torch.Generator().manual_seed(3)
    x = STRIDED[view](torch.randn(6, 40, 264, generator=gen).to(dtype).to(cuda))
    width = x.shape[-1]
    w, b = (torch.randn(width, generator=gen).to(dtype).to(cuda) for _ in range(2))
    g = torch.randn(x.shape, generator=gen).to(dtype).to(cuda)
    leaves = [x.detach().requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True)]
    y = layer_norm(*leaves)
    got = (y, *torch.autograd.grad(y, leaves, g))
    flat = [t.detach().reshape(-1, width) for t in (x, g)]
    for t, (exact, lost) in zip(got, norm_with_bounds(flat[0], w.detach(), b.detach(), flat[1], 1e-5)):
        check(t.reshape(exact.shape), exact, lost)


def test_norm_of_rows_far_from_zero(cuda):
    """The variance is taken about the mean: an offset of 3000 spreads costs 3000 roundings of x and no more."""
    gen = torch.Generator().manual_seed(5)
    for width in (200, 2048, 40000):
        x = (3000 + torch.randn(9, width, generator=gen)).to(cuda)
        w = torch.ones(width, device=cuda)
        check_norm(x, w, None, torch.randn(9, width, generator=gen).to(cuda))


def test_norm_of_constant_rows_zeros_and_nan(cuda):
    w, b = torch.full((128,), 2.0, device=cuda), torch.full((128,), 0.25, device=cuda)
    x = torch.zeros(4, 128, device=cuda)
    x[1] = 7.0
    x[2, 5] = float("nan")
    x[3, 5] = float("inf")
    y = layer_norm(x, w, b)
    assert torch.equal(y[:2], torch.full_like(y[:2], 0.25)) and y[2:].isnan().all()


def test_norm_without_rows_and_of_one_vector(cuda):
    w = torch.randn(16, device=cuda, requires_grad=True)
    b = torch.randn(16, device=cuda, requires_grad=True)
    x = torch.randn(0, 16, device=cuda, requires_grad=True)
    y = layer_norm(x, w, b)
    grads = torch.autograd.grad(y.sum(), (x, w, b))
    assert y.shape == (0, 16) and grads[0].shape == (0, 16) and not grads[1].any() and not grads[2].any()
    one = torch.randn(16, device=cuda)
    assert torch.equal(layer_norm(one, w, b), layer_norm(one[None], w, b)[0])
    assert layer_norm(torch.randn(2, 0, 3, 16, device=cuda), w, b).shape == (2, 0, 3, 16)


def test_norm_gives_only_the_gradients_that_are_wanted(cuda):
    x, w, b, g = norm_case(300, 520, torch.bfloat16, True, True, cuda)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    want = torch.autograd.grad(layer_norm(*leaves), leaves, g)
    for k in range(3):
        inputs = [t.clone().requires_grad_(i == k) for i, t in enumerate((x, w, b))]
        got, = torch.autograd.grad(layer_norm(*inputs), inputs[k], g)
        assert torch.equal(got, want[k])


def test_norm_gradients_against_differences(cuda):
    x, w, b, g = norm_case(3, 20, torch.float32, False, True, cuda)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(layer_norm(*leaves), leaves, g)
    for k, leaf in enumerate(leaves):
        flat = leaf.detach().view(-1)
        for i in range(0, flat.numel(), 7):
            step = 2.0 ** -7
            sides = []
            for sign in (1, -1):
                moved = [t.detach().clone() for t in leaves]
                moved[k].view(-1)[i] += sign * step
                sides.append((plain.layer_norm(*moved) * g.double()).sum().item())
            # the formula in 64 bits: what is left is the third derivative's, some units times step^2
            assert abs((sides[0] - sides[1]) / (2 * step) - grads[k].view(-1)[i].item()) < 40 * step ** 2


# ------------------------------------------------------------------- dropout

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1,), (3,), (7,), (8,), (33,), (5, 4, 3), (1000, 1021), (64, 2048)])
def test_dropout_and_gradients_match_the_plain_form(shape, dtype, cuda):
    gen = torch.Generator().manual_seed(len(shape) + shape[0])
    x, r, g = (torch.randn(shape, generator=gen).to(dtype).to(cuda) for _ in range(3))
    for probability, seed, site, step in ((0.1, 7, 3, 11), (0.5, 2 ** 64 - 1, 0, 2 ** 63), (0.0, 5, 1, 1), (1.0, 5, 1, 1)):
        for residual in (None, r):
            leaves = [t.clone().requires_grad_(True) for t in (x, residual) if t is not None]
            y = dropout(leaves[0], probability, seed=seed, site=site, step=step, residual=None if residual is None else leaves[1])
            # the scale, the product and the sum: 3 roundings of the scaled value
            scaled = x.double().abs() * (2 if probability < 1 else 0)
            check(y, plain.dropout(x, probability, seed, site, step, residual), 3 * EPS * scaled)
            grads = torch.autograd.grad(y, leaves, g)
            check(grads[0], plain.dropout(g, probability, seed, site, step), 2 * EPS * g.double().abs() * 2)
            if residual is not None:
                assert torch.equal(grads[1], g)


def test_dropout_share_and_mean(cuda):
    """Of n values about p n are dropped: five standard deviations of the binomial, for 300 sites in turn."""
    x = torch.ones(1 << 16, device=cuda)
    for p in (0.1, 0.3):
        shares = torch.stack([(dropout(x, p, seed=9, site=site) == 0).double().mean() for site in range(300)])
        exact = int(p * 65536 + 0.5) / 65536
        spread = (exact * (1 - exact) / x.numel()) ** 0.5
        assert (shares - exact).abs().max().item() < 5 * spread
        assert (shares.mean() - exact).abs().item() < 5 * spread / 300 ** 0.5


def test_dropout_of_strided_and_offset_values(cuda):
    base = torch.randn(40, 70, device=cuda)
    for x in (base.T, base[:, 3:], base[::3], base.flatten()[1:], base[0, 0].expand(9, 9)):
        assert torch.equal(dropout(x, 0.4, seed=1), dropout(x.contiguous().clone(), 0.4, seed=1))
        assert torch.equal(dropout(x.contiguous().clone(), 0.4, seed=1, residual=x), dropout(x, 0.4, seed=1, residual=x.contiguous()))


def test_dropout_drops_infinities_and_nan(cuda):
    x = torch.full((4096,), float("nan"), device=cuda)
    x[::2] = float("inf")
    y = dropout(x, 0.5, seed=3)
    kept = torch.from_numpy(plain.dropout_lanes(0, 4096, 3, 0, 0) >= 32768).to(cuda)
    assert (y[~kept] == 0).all() and torch.equal(y[kept].isnan(), x[kept].isnan()) and torch.equal(y[kept].isinf(), x[kept].isinf())
    r = torch.randn(4096, device=cuda)
    assert torch.equal(dropout(x, 1.0, seed=3, residual=r), r)


def test_dropout_positions_past_32_bits(cuda):
    """4.3 thousand million values: the position is 64 bits wide, in whole packets and behind the last."""
    count = (1 << 32) + 4099
    x = torch.ones(count, dtype=torch.bfloat16, device=cuda)
    y = dropout(x, 0.25, seed=21, site=2, step=1)
    del x
    for first in (0, (1 << 31) - 64, (1 << 32) - 64, count - 5000):
        n = min(5000, count - first)
        want = torch.from_numpy(plain.dropout_lanes(first, n, 21, 2, 1) >= 16384).to(cuda)
        assert torch.equal(y[first:first + n] != 0, want)
    del y
    torch.cuda.empty_cache()


def test_dropout_step_on_the_device(cuda):
    x = torch.randn(1000, device=cuda, requires_grad=True)
    step = torch.tensor(12, device=cuda)
    y = dropout(x, 0.3, seed=1, step=step)
    assert torch.equal(y, dropout(x, 0.3, seed=1, step=12))
    grad, = torch.autograd.grad(y, x, torch.ones_like(y), retain_graph=True)
    assert torch.equal(grad != 0, y != 0)
    step += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, x, torch.ones_like(y))


def test_dropout_is_linear_to_every_order(cuda):
    x = torch.randn(100, device=cuda, requires_grad=True)
    g = torch.randn(100, device=cuda, requires_grad=True)
    grad, = torch.autograd.grad(dropout(x, 0.3, seed=1), x, g, create_graph=True)
    again, = torch.autograd.grad(grad, g, torch.ones_like(g))
    assert torch.equal(again, dropout(torch.ones(100, device=cuda), 0.3, seed=1))


def test_layer_norm_rows_past_32_bits(cuda):
    """4.3 thousand million entries. Two results of the same rows are each within a rounding and fp32's
    errors of the formula, so they differ by no more than three roundings, 3 * 2^-8 of the norm."""
    rows = (1 << 26) + 777
    g = torch.Generator(device=cuda).manual_seed(4)
    x = torch.empty(rows, 64, dtype=torch.bfloat16, device=cuda).normal_(generator=g)
    weight, bias = torch.randn(2, 64, generator=g, device=cuda)
    y = layer_norm(x.requires_grad_(True), weight, bias)
    dx, = torch.autograd.grad(y, x, y.detach())
    y, x = y.detach(), x.detach()
    for first in (0, (1 << 25) - 100, rows - 3000):
        part = x[first:first + 3000].clone().requires_grad_(True)
        want = layer_norm(part, weight, bias)
        grad, = torch.autograd.grad(want, part, y[first:first + 3000].clone())
        for got, w in ((y[first:first + 3000], want), (dx[first:first + 3000], grad)):
            assert (got.double() - w.double()).norm() <= 3 * 2.0 ** -8 * w.double().norm()
    del x, y, dx
    torch.cuda.empty_cache()
