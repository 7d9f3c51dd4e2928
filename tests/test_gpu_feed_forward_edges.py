"""Corners of the feed-forward sub-layer's operators on the GPU: values at the ends of their range, every plan of the
norm's kernels, buffers of exactly the size that the C entries ask for, calls on several streams at once."""
from __future__ import annotations

import pytest
import torch

from koemi_5hom_b200 import _native
from koemi_5hom_b200.cuda_kernels.core import dropout, layer_norm
from koemi_5hom_b200.cuda_kernels.dense import gated_feed_forward

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def normal(cuda, seed=0):
    g = torch.Generator().manual_seed(seed)
    return lambda *shape, scale=1.0, dtype=torch.float32: (scale * torch.randn(*shape, generator=g)).to(dtype).to(cuda)


# ---------------------------------------------------------------- layer norm

@pytest.mark.parametrize("rows", [5, 1500])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width,exponent,eps", [(33, 120, 1e-5), (96, 120, 1e-5), (40, 120, 1e-5), (1021, 110, 1e-12), (1032, 110, 1e-12),
                                                (2312, 110, 1e-12), (16384, 110, 1e-12), (33000, 110, 1e-12)])
def test_norm_of_large_constant_rows(width, exponent, eps, dtype, rows, cuda):
    """The mean is exact (a power of two, at widths n with fl(fl(1 / n) n) = 1), so u is 0, y is b and dw is 0 to the bit,
    and dx = (a - mean(a)) / sqrt(eps). Mean times 1 / sqrt(eps) is past fp32's range: nothing may form it."""
    new = normal(cuda, width)
    x = torch.full((rows, width), 2.0 ** exponent, dtype=dtype, device=cuda, requires_grad=True)
    w, b = (new(width).requires_grad_(True) for _ in range(2))
    g = new(rows, width, dtype=dtype)
    y = layer_norm(x, w, b, eps=eps)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), g)
    assert torch.equal(y, b.to(dtype).expand_as(y)) and not dw.any()
    # a sum over a row is at most width / 1024 + 40 additions deep, over rows rows / 148 + 100; the rest: 12 roundings
    deep, down = (width / 1024 + 40) * EPS, (rows / 148 + 100) * EPS
    a = g.double() * w.detach().double()
    mean, inverse = a.mean(-1, keepdim=True), eps ** -0.5
    want = inverse * (a - mean)
    allowed = inverse * (2 * deep * a.abs().mean(-1, keepdim=True) + (deep + 12 * EPS) * (a.abs() + mean.abs()))
    assert ((dx.double() - want).abs() <= U[dtype] * 1.0001 * want.abs() + allowed).all()
    assert ((db.double() - g.double().sum(0)).abs() <= EPS * db.double().abs() + 2 * down * g.double().abs().sum(0)).all()


# -------------------------------------------------------- torch's transforms

def test_vmap(cuda):
    """Refused where samples would share a mask; else the samples' own results."""
    new = normal(cuda)
    x, w, b = new(5, 40, 64), new(64), new(64)
    wg, wv, wo = new(48, 64), new(48, 64), new(64, 48)
    assert torch.equal(torch.vmap(lambda t: layer_norm(t, w, b))(x), torch.stack([layer_norm(t, w, b) for t in x]))
    assert torch.equal(torch.vmap(lambda t: gated_feed_forward(t, wg, wv, wo))(x), torch.stack([gated_feed_forward(t, wg, wv, wo) for t in x]))
    for call in (lambda t: dropout(t, 0.1, seed=1), lambda t: dropout(x[0], 0.1, seed=1, residual=t)):
        with pytest.raises(NotImplementedError, match="vmap"):
            torch.vmap(call)(x)


# ---------------------------------------------------------------- memory

def test_block_takes_no_memory_that_it_does_not_use(cuda):
    """A training pass of aligned bf16: the forward leaves y and what the backward needs (h in 2 bytes a hidden value,
    two slopes in 4), the backward takes what the query asks for operands that are read as they lie; a megabyte for the allocator."""
    rows, width, hidden = 16384, 512, 1024
    new = normal(cuda)
    leaves = [new(*shape, dtype=torch.bfloat16).requires_grad_(True) for shape in ((rows, width), (hidden, width), (hidden, width), (width, hidden))]
    grad = new(rows, width, dtype=torch.bfloat16)

    def peak(call):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        result = call()
        torch.cuda.synchronize()
        return result, torch.cuda.max_memory_allocated() - before

    y, forward = peak(lambda: gated_feed_forward(*leaves))
    assert forward <= 2 * rows * width + 10 * rows * hidden + 2 ** 20
    results, backward = peak(lambda: torch.autograd.grad(y, leaves, grad))
    ask = lambda bits: _native.library().koemi_dense_gated_feed_forward_workspace(rows, width, hidden, width, _native.BF16, bits)  # noqa: E731
    assert backward <= sum(2 * t.numel() for t in leaves) + ask(1 | 4) + 2 ** 20 and ask(1 | 4) <= ask(1) - 4 * rows * width
