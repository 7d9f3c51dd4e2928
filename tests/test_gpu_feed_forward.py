"""The gated feed-forward block on the GPU against plain 64-bit forms (oracle/feed_forward.py).

On integers that every type holds, with gates so large that silu(p) = p, every
product and sum is exact: there the results are equal bit for bit, whatever the
tiles. On ordinary values an entry is held to what its terms' roundings may add up
to, and each result as a whole to a few roundings.
"""
from __future__ import annotations

import pytest
import torch

from koemi_5hom_b200.cuda_kernels.dense import gated_feed_forward
from oracle import feed_forward as plain

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -120, torch.bfloat16: 2.0 ** -120, torch.float16: 2.0 ** -25}  # fp16: half the subnormal spacing
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
NAMES = ("y", "dx", "dwg", "dwv", "dwo", "dbg", "dbv", "dbo")

# rows, width, hidden, out
SHAPES = [(1, 1, 1, 1), (1, 8, 8, 8), (2, 15, 30, 7), (7, 64, 64, 64), (3, 65, 127, 33), (4, 512, 264, 100), (8, 300, 1040, 56),
          (9, 72, 40, 64), (5, 1000, 2000, 1000), (2, 4100, 260, 4100), (127, 200, 129, 72), (128, 128, 256, 128),
          (129, 72, 520, 515), (300, 515, 1030, 515), (1000, 96, 40, 264), (1, 2048, 4096, 2048), (64, 1000, 2000, 1000),
          (256, 2048, 4096, 2048), (5000, 64, 136, 40), (777, 1024, 384, 1032)]


def run(arguments, grad):
    """y and the gradients of all that is not None, in the order of NAMES."""
    leaves = [None if t is None else t.detach().requires_grad_(True) for t in arguments]
    y = gated_feed_forward(*leaves[:4], gate_bias=leaves[4], value_bias=leaves[5], output_bias=leaves[6])
    given = [t for t in leaves if t is not None]
    grads = iter(torch.autograd.grad(y, given, grad))
    with torch.no_grad():
        again = gated_feed_forward(*arguments[:4], gate_bias=arguments[4], value_bias=arguments[5], output_bias=arguments[6])
    assert torch.equal(again.isnan(), y.isnan()) and torch.equal(again.nan_to_num(), y.nan_to_num())
    return [y.detach()] + [None if t is None else next(grads) for t in leaves]


# ------------------------------------------------------------ exact on integers

def integers(rows, width, hidden, out, dtype, cuda, bias=True, seed=0):
    """Few nonzero entries a row, so that p stays near 64 and all sums stay small."""
    g = torch.Generator().manual_seed(seed + rows + 3 * width + 5 * hidden + 7 * out)

    def sparse(a, b, each, most=1):
        density = min(1.0, each / b)
        values = torch.randint(-most, most + 1, (a, b), generator=g)
        return (values * (torch.rand(a, b, generator=g) < density)).to(dtype).to(cuda)

    x, wg, wv, wo = sparse(rows, width, 12, 2), sparse(hidden, width, 12), sparse(hidden, width, 6), sparse(out, hidden, 8)
    bg = (64 + torch.randint(-3, 4, (hidden,), generator=g)).to(dtype).to(cuda)
    bv, bo = (torch.randint(-2, 3, (n,), generator=g).to(dtype).to(cuda) if bias else None for n in (hidden, out))
    return (x, wg, wv, wo, bg, bv, bo), sparse(rows, out, 6)


def rounded_form(arguments, grad):
    """The formulas in 64 bits with the roundings of the type where the block has them."""
    dtype = arguments[0].dtype
    x, wg, wv, wo, bg, bv, bo = (None if t is None else t.double() for t in arguments)
    g = grad.double()
    keep = (lambda t: t) if dtype == torch.float32 else (lambda t: t.to(dtype).double())
    p, q = x @ wg.T + bg, x @ wv.T + (0 if bv is None else bv)
    assert p.min().item() > 24  # 1 / (1 + exp(-p)) is 1 in fp32
    h = keep(p * q)
    y = h @ wo.T + (0 if bo is None else bo)
    dh = g @ wo
    dp, dq = keep(dh * q), keep(dh * p)
    results = [y, dp @ wg + dq @ wv, dp.T @ x, dq.T @ x, g.T @ h, dp.sum(0), dq.sum(0), g.sum(0)]
    assert max(t.abs().max().item() for t in results) < 2 ** 24  # exact in fp32, in whatever order
    return [t.to(dtype) for t in results]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_integers_are_exact(shape, dtype, cuda):
    arguments, grad = integers(*shape, dtype, cuda)
    for name, got, want in zip(NAMES, run(arguments, grad), rounded_form(arguments, grad)):
        assert got.dtype == dtype and torch.equal(got, want), f"{name}: {(got != want).sum().item()} of {got.numel()} differ"


@pytest.mark.parametrize("dtype", DTYPES)
def test_integers_without_two_biases(dtype, cuda):
    arguments, grad = integers(200, 136, 264, 96, dtype, cuda, bias=False)
    for got, want in zip(run(arguments, grad), rounded_form(arguments, grad)):
        assert got is None or torch.equal(got, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(8192, 512, 1024, 512), (20000, 256, 512, 264), (3000, 4096, 640, 4096)], ids=str)
def test_integers_of_large_problems(shape, dtype, cuda):
    """More tiles than the GPU holds at once, long sums, several bands."""
    arguments, grad = integers(*shape, dtype, cuda)
    for name, got, want in zip(NAMES, run(arguments, grad), rounded_form(arguments, grad)):
        assert torch.equal(got, want), f"{name}: {(got != want).sum().item()} of {got.numel()} differ"


# ------------------------------------------------------------- ordinary values

def ordinary(rows, width, hidden, out, dtype, cuda, bias, seed=0):
    g = torch.Generator().manual_seed(seed + rows + width + hidden)

    def normal(*shape, scale=1.0):
        return (scale * torch.randn(*shape, generator=g)).to(dtype).to(cuda)

    arguments = [normal(rows, width), normal(hidden, width, scale=1.5 * width ** -0.5), normal(hidden, width, scale=width ** -0.5),
                 normal(out, hidden, scale=hidden ** -0.5)]
    arguments += [normal(hidden, scale=0.5), normal(hidden, scale=0.5), normal(out, scale=0.5)] if bias else [None] * 3
    return arguments, normal(rows, out)


def form_with_bounds(arguments, grad):
    """64-bit results and what the block may lose of each, entry by entry.

    A sum of k products on the tensor cores rounds (or cuts off) its running
    value a few times every 16 products: k / 4 + 32 EPS of the sum of magnitudes, six times as
    many products in fp32. |silu'| <= 1.1, |silu''| <= 0.5; exponentials and
    quotients lose 16 EPS (1 + |p|). u: the roundings of the type between the products.
    """
    dtype = arguments[0].dtype
    x, wg, wv, wo, bg, bv, bo = (None if t is None else t.double() for t in arguments)
    g = grad.double()
    u = 0.0 if dtype == torch.float32 else U[dtype] * 1.0001
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    times = 6 if dtype == torch.float32 else 1
    deep = lambda k: (times * k / 4 + 32) * EPS  # noqa: E731
    plus = lambda t, b: t if b is None else t + b  # noqa: E731
    p, q = plus(x @ wg.T, bg), plus(x @ wv.T, bv)
    p_lost = deep(x.shape[1]) * plus(x.abs() @ wg.abs().T, None if bg is None else bg.abs())
    q_lost = deep(x.shape[1]) * plus(x.abs() @ wv.abs().T, None if bv is None else bv.abs())
    s = torch.sigmoid(p)
    act, slope, curve = p * s, s * (1 + p * (1 - s)), 16 * EPS * (1 + p.abs())
    h = act * q
    h_lost = 1.1 * p_lost * q.abs() + act.abs() * q_lost + curve * h.abs() + 1.1 * p_lost * q_lost
    h_lost = h_lost + u * (h.abs() + h_lost) + tiny
    y = plus(h @ wo.T, bo)
    y_lost = h_lost @ wo.abs().T + deep(h.shape[1]) * plus(h.abs() @ wo.abs().T, None if bo is None else bo.abs())
    dh, dh_lost = g @ wo, deep(g.shape[1]) * (g.abs() @ wo.abs())
    dq = dh * act
    dq_lost = dh_lost * act.abs() + dh.abs() * 1.1 * p_lost + 2 * curve * dq.abs()
    dp = dh * q * slope
    dp_lost = dh_lost * (q * slope).abs() + dh.abs() * (1.1 * q_lost + 0.5 * q.abs() * p_lost + 0.5 * p_lost * q_lost) + 2 * curve * (dh * q).abs()
    dq_lost, dp_lost = (lost * (1 + u) + u * t.abs() + tiny for lost, t in ((dq_lost, dq), (dp_lost, dp)))
    rows = deep(x.shape[0])
    dx_lost = dp_lost @ wg.abs() + dq_lost @ wv.abs() + deep(2 * h.shape[1]) * (dp.abs() @ wg.abs() + dq.abs() @ wv.abs())
    results = [(y, y_lost), (dp @ wg + dq @ wv, dx_lost), (dp.T @ x, dp_lost.T @ x.abs() + rows * (dp.abs().T @ x.abs())),
               (dq.T @ x, dq_lost.T @ x.abs() + rows * (dq.abs().T @ x.abs())),
               (g.T @ h, g.abs().T @ h_lost + rows * (g.abs().T @ h.abs())),
               (dp.sum(0), dp_lost.sum(0) + rows * dp.abs().sum(0)), (dq.sum(0), dq_lost.sum(0) + rows * dq.abs().sum(0)),
               (g.sum(0), rows * g.abs().sum(0))]
    return results


def check_ordinary(arguments, grad):
    dtype = arguments[0].dtype
    for name, got, (exact, lost) in zip(NAMES, run(arguments, grad), form_with_bounds(arguments, grad)):
        if got is None:
            continue
        off = got.double() - exact
        over = off.abs() - (U[dtype] * 1.0001 * exact.abs() + lost + TINY[dtype])
        assert got.shape == exact.shape and over.max().item() <= 0, f"{name} is off by {over.max().item()} more than allowed"
        if exact.numel() > 1000:
            # As a whole: an error is a root mean square of at most U / sqrt(3) a rounding, and no result has gone
            # through more than two of them (h, dp or dq, and its own): 0.82 U in all. A token's gradients may hang on
            # few dp: U sqrt(3). fp32's sums add their own, of terms of one size.
            most = 3 ** 0.5 * U[dtype] if dtype != torch.float32 else 2e-6
            assert off.norm().item() <= most * exact.norm().item(), f"{name}: {off.norm().item() / exact.norm().item()}"


@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_block_and_gradients_match_the_plain_form(shape, dtype, bias, cuda):
    check_ordinary(*ordinary(*shape, dtype, cuda, bias))


def test_gradients_against_differences(cuda):
    arguments, grad = ordinary(5, 24, 40, 16, torch.float32, cuda, True)
    got = run(arguments, grad)[1:]
    step = 2.0 ** -7
    for k, leaf in enumerate(arguments):
        for i in range(0, leaf.numel(), max(1, leaf.numel() // 9)):
            sides = []
            for sign in (1, -1):
                moved = [t.clone() for t in arguments]
                moved[k].view(-1)[i] += sign * step
                sides.append((plain.gated_feed_forward(*moved) * grad.double()).sum().item())
            # the formula in 64 bits: what is left is the third derivative's, some tens of units times step^2
            assert abs((sides[0] - sides[1]) / (2 * step) - got[k].view(-1)[i].item()) < 60 * step ** 2


@pytest.mark.parametrize("dtype", DTYPES)
def test_values_of_other_shapes_strides_and_starts(dtype, cuda):
    (x, *rest), grad = ordinary(60, 64, 128, 64, dtype, cuda, True)
    weights, biases = rest[:3], dict(zip(("gate_bias", "value_bias", "output_bias"), rest[3:]))
    want = gated_feed_forward(x, *weights, **biases)
    wide = torch.randn(60, 200, device=cuda).to(dtype)
    wide[:, 8:72] = x
    odd = torch.randn(60, 201, device=cuda).to(dtype)
    odd[:, 3:67] = x
    flat = torch.cat((x.new_zeros(1), x.flatten()))[1:].view(60, 64)
    for view in (x.view(3, 4, 5, 64), wide[:, 8:72], odd[:, 3:67], flat, x.T.contiguous().T, x.view(3, 20, 64).transpose(0, 1).contiguous().transpose(0, 1)):
        assert torch.equal(gated_feed_forward(view, *weights, **biases).reshape(60, 64), want)
        leaf = view.detach().requires_grad_(True)
        got, = torch.autograd.grad(gated_feed_forward(leaf, *weights, **biases), leaf, grad.view(*view.shape[:-1], 64))
        base = x.clone().requires_grad_(True)
        expected, = torch.autograd.grad(gated_feed_forward(base, *weights, **biases), base, grad)
        assert torch.equal(got.reshape(60, 64), expected)
    transposed = [t.T.contiguous().T for t in weights]
    off = [torch.cat((t.new_zeros(1), t.flatten()))[1:].view(t.shape) for t in weights]
    for other in (transposed, off):
        assert torch.equal(gated_feed_forward(x, *other, **biases), want)
    assert torch.equal(gated_feed_forward(x[7], *weights, **biases), gated_feed_forward(x[7:8], *weights, **biases)[0])
    same = x[:1].expand(60, 64)
    assert torch.equal(gated_feed_forward(same, *weights, **biases), gated_feed_forward(same.contiguous(), *weights, **biases))


def test_only_the_gradients_that_are_wanted(cuda):
    arguments, grad = ordinary(300, 72, 136, 40, torch.bfloat16, cuda, True)
    want = run(arguments, grad)[1:]
    for k in range(7):
        leaves = [t.detach().requires_grad_(i == k) for i, t in enumerate(arguments)]
        y = gated_feed_forward(*leaves[:4], gate_bias=leaves[4], value_bias=leaves[5], output_bias=leaves[6])
        assert torch.equal(torch.autograd.grad(y, leaves[k], grad)[0], want[k])


def test_no_rows(cuda):
    arguments, _ = ordinary(1, 16, 24, 8, torch.bfloat16, cuda, True)
    arguments[0] = arguments[0][:0]
    y, *grads = run(arguments, torch.zeros(0, 8, dtype=torch.bfloat16, device=cuda))
    assert y.shape == (0, 8) and grads[0].shape == (0, 16) and not any(g.any() for g in grads[1:])


def test_rows_are_independent_of_what_is_beside_them(cuda):
    """A NaN row gives NaN in its own row of y and dx, and nowhere else in them."""
    for dtype in DTYPES:
        arguments, grad = ordinary(200, 64, 128, 64, dtype, cuda, False)
        clean = run(arguments, grad)
        arguments[0][131] = float("nan")
        dirty = run(arguments, grad)
        keep = torch.arange(200, device=cuda) != 131
        assert torch.equal(dirty[0][keep], clean[0][keep]) and torch.equal(dirty[1][keep], clean[1][keep])
        assert dirty[0][131].isnan().all() and dirty[1][131].isnan().all() and dirty[2].isnan().all()


def test_large_and_small_fp32_values(cuda):
    """fp32 keeps its precision at every scale that its products stay in."""
    for scale in (2.0 ** -40, 2.0 ** 30):
        arguments, grad = ordinary(100, 96, 64, 80, torch.float32, cuda, False)
        arguments[0] = arguments[0] * scale
        arguments[1], arguments[2] = arguments[1] / scale, arguments[2] / scale
        check_ordinary(arguments, grad)


@pytest.mark.parametrize("rows", [2, 3, 4, 8, 9])
@pytest.mark.parametrize("dtype", DTYPES)
def test_few_rows_are_independent_of_what_is_beside_them(rows, dtype, cuda):
    for width in (64, 33):
        arguments, _ = ordinary(rows, width, 40, 24, dtype, cuda, True)
        weights, biases = arguments[1:4], dict(gate_bias=arguments[4], value_bias=arguments[5], output_bias=arguments[6])
        clean = gated_feed_forward(arguments[0], *weights, **biases)
        arguments[0][rows - 1, width - 1] = float("nan")
        dirty = gated_feed_forward(arguments[0], *weights, **biases)
        assert torch.equal(dirty[:-1], clean[:-1]) and dirty[-1].isnan().all()


def test_rows_past_32_bits(cuda):
    """x, dx, y and dy of 4.3 thousand million entries. Two results of the same rows are each within three
    roundings of the formula, so they differ by no more than six, 6 U of the norm."""
    rows, limit = (1 << 26) + 777, 6 * U[torch.bfloat16]
    g = torch.Generator(device=cuda).manual_seed(3)
    x = torch.empty(rows, 64, dtype=torch.bfloat16, device=cuda).normal_(generator=g)
    weights = [(torch.randn(a, b, generator=g, device=cuda) / 8).bfloat16() for a, b in ((16, 64), (16, 64), (64, 16))]
    y = gated_feed_forward(x.requires_grad_(True), *weights)
    dx, = torch.autograd.grad(y, x, x.detach())
    y, x = y.detach(), x.detach()
    for first in (0, (1 << 25) - 100, rows - 3000):
        part = x[first:first + 3000].clone().requires_grad_(True)
        want = gated_feed_forward(part, *weights)
        grad, = torch.autograd.grad(want, part, part.detach())
        for got, w in ((y[first:first + 3000], want), (dx[first:first + 3000], grad)):
            assert (got.double() - w.double()).norm() <= limit * w.double().norm()
    del x, y, dx
    torch.cuda.empty_cache()
