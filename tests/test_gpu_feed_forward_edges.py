"""Corners of the feed-forward sub-layer's operators on the GPU: values at the ends of their range, every plan of the
norm's kernels, buffers of exactly the size that the C entries ask for, calls on several streams at once."""
from __future__ import annotations

import threading

import pytest
import torch
from test_gpu_feed_forward import form_with_bounds, ordinary, run
from test_gpu_layer_norm import check_norm, norm_case

from koemi_5hom_b200 import _native
from koemi_5hom_b200.cuda_kernels.core import dropout, layer_norm
from koemi_5hom_b200.cuda_kernels.dense import gated_feed_forward
from oracle import feed_forward as plain

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


@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("wide", [True, False])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [16, 128, 256, 260, 512, 520, 4096, 8192])
def test_norm_of_many_rows_in_every_plan(width, dtype, wide, bias, cuda):
    """More rows than 8 an SM, where a thread takes several packets: 1, 8, 16 and 32 lanes a row, the first widths that
    take a CTA a row, and long rows; weights and biases of either type."""
    check_norm(*norm_case(1300, width, dtype, wide, bias, cuda))


# ---------------------------------------------------------- the gated block

def test_small_fp16_gradients(cuda):
    """A loss that is not scaled: dp and dq reach into fp16's subnormal numbers and past their end. Every gradient is
    what the formula gives with 2^-25 lost of each of them; scaled by 2^14 it keeps its digits."""
    arguments, grad = ordinary(300, 96, 136, 72, torch.float16, cuda, True)
    grad = grad * 2.0 ** -16
    for got, (exact, lost) in zip(run(arguments, grad), form_with_bounds(arguments, grad)):
        over = (got.double() - exact).abs() - (U[torch.float16] * 1.0001 * exact.abs() + lost + 2.0 ** -25)
        assert over.max().item() <= 0
    scaled = grad * 2.0 ** 14  # exact
    for got, (exact, _) in list(zip(run(arguments, scaled), form_with_bounds(arguments, scaled)))[1:]:
        assert (got.double() - exact).norm() <= 3 ** 0.5 * U[torch.float16] * exact.norm()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_weight_gradients_of_long_sums(dtype, cuda):
    """A million rows whose terms are all positive, so that nothing of the sums' own errors cancels. An entry goes through
    two roundings (h, dp or dq, and its own); an accumulator is cut off at its last place, 2^-23 of it, once in 16 rows,
    and with few tiles K is in 8 parts at least: 2^20 / 16 / 8 steps, 2^-10 in all."""
    rows, width, hidden, out = 1 << 20, 64, 48, 40
    g = torch.Generator(device=cuda).manual_seed(8)
    uniform = lambda scale, *shape: (scale * (0.5 + 0.5 * torch.rand(shape, generator=g, device=cuda))).to(dtype).requires_grad_(True)  # noqa: E731
    leaves = [uniform(1, rows, width), uniform(1 / width, hidden, width), uniform(1 / width, hidden, width), uniform(1 / out, out, hidden),
              uniform(0.1, hidden), uniform(0.1, hidden), uniform(0.1, out)]
    grad = uniform(2.0 ** -8, rows, out).detach()  # the sums stay in fp16's range, dp and dq in its normal numbers
    names = ("gate_bias", "value_bias", "output_bias")
    got = torch.autograd.grad(gated_feed_forward(*leaves[:4], **dict(zip(names, leaves[4:]))), leaves[1:], grad)
    exact = [t.detach().double().requires_grad_(True) for t in leaves]
    want = torch.autograd.grad(plain.gated_feed_forward(*exact), exact[1:], grad.double())
    for a, b in zip(got, want):
        assert b.min().item() > 0 and ((a.double() - b).abs() <= (2.01 * U[dtype] + 2.0 ** -10) * b).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("chunk", [9, 16, 32, 144])
def test_a_batch_is_its_parts_on_tensor_cores(chunk, dtype, cuda):
    """9 rows and more take the tensor cores in every type, their K cut by the number of rows: parts of a batch agree
    with the whole to what two results may differ from the formula, 3^0.5 U each of the norm (fp32: 2^-19 for the sums)."""
    (x, *weights), _ = ordinary(288, 1024, 2048, 512, dtype, cuda, True)
    biases = dict(zip(("gate_bias", "value_bias", "output_bias"), weights[3:]))
    call = lambda t: gated_feed_forward(t, *weights[:3], **biases)  # noqa: E731
    whole, parts = call(x).double(), torch.cat([call(t) for t in x.split(chunk)]).double()
    most = 2.0 ** -19 if dtype == torch.float32 else 2 * 3 ** 0.5 * U[dtype]
    assert (whole - parts).norm() <= most * whole.norm()


# ------------------------------------------------- buffers of exactly their size

GUARD = 1024


class Buffers:
    """Device buffers of exactly the bytes asked for, between bytes that nothing may touch."""

    def __init__(self, device):
        self.device, self.all = device, []

    def new(self, nbytes, shift=0):
        buffer = torch.full((nbytes + 2 * GUARD,), 0xA5, dtype=torch.uint8, device=self.device)
        self.all.append((buffer, GUARD + shift, nbytes))
        return buffer.data_ptr() + GUARD + shift

    def values(self, index, dtype, *shape):
        buffer, start, nbytes = self.all[index]
        return buffer[start:start + nbytes].clone().view(dtype).view(shape)

    def check(self):
        torch.cuda.synchronize()
        for buffer, start, nbytes in self.all:
            assert (buffer[:start] == 0xA5).all() and (buffer[start + nbytes:] == 0xA5).all()


def stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.fixture
def buffers(cuda):
    _native.ensure_device(cuda)
    return Buffers(cuda)


FEW = [(rows, dtype, shape) for dtype in DTYPES for rows in ((1, 3, 8) if dtype == torch.float32 else (1, 2, 4))
       for shape in ((64, 72, 40), (33, 77, 21), (2048, 264, 24))]


@pytest.mark.parametrize("keeps", [True, False])
@pytest.mark.parametrize("rows,dtype,shape", FEW + [(9, torch.float32, (40, 264, 65)), (257, torch.float16, (64, 128, 200))], ids=str)
def test_block_writes_its_buffers_and_no_more(rows, dtype, shape, keeps, buffers, cuda):
    width, hidden, out = shape
    lib, code, new = _native.library(), _native.dtype_code(dtype), normal(cuda, rows)
    x, wg, wv, wo, grad = (new(*s, scale=0.3, dtype=dtype) for s in ((rows, width), (hidden, width), (hidden, width), (out, hidden), (rows, out)))
    ask = lambda bits: lib.koemi_dense_gated_feed_forward_workspace(rows, width, hidden, out, code, bits | 4)  # noqa: E731
    size, kept_size = x.element_size(), lib.koemi_dense_gated_feed_forward_kept(rows, hidden, code)
    y, kept = buffers.new(rows * out * size), buffers.new(kept_size) if keeps else None
    room = ask(2 * keeps)
    operands = (x.data_ptr(), width, wg.data_ptr(), wv.data_ptr(), wo.data_ptr())
    assert lib.koemi_dense_gated_feed_forward_forward(*operands, None, None, None, y, kept, kept_size if keeps else 0, rows, width, hidden, out, code,
                                                      buffers.new(room), room, stream()) == 0
    assert torch.equal(buffers.values(0, dtype, rows, out), gated_feed_forward(x, wg, wv, wo))
    if keeps:
        counts = (rows * width, hidden * width, hidden * width, out * hidden, hidden, hidden, out)
        first, room = len(buffers.all), ask(1)
        grads = [buffers.new(n * size) for n in counts]
        assert lib.koemi_dense_gated_feed_forward_backward(*operands, kept, kept_size, grad.data_ptr(), *grads, rows, width, hidden, out, code,
                                                           buffers.new(room), room, stream()) == 0
        leaves = [t.requires_grad_(True) for t in (x, wg, wv, wo)]
        for k, want in enumerate(torch.autograd.grad(gated_feed_forward(*leaves), leaves, grad)):
            assert torch.equal(buffers.values(first + k, dtype, *want.shape), want)
    buffers.check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width", [(5, 64), (2001, 33), (2001, 96), (5, 1032), (1300, 1021), (1300, 2048), (3, 16384), (300, 16384), (3, 33000)])
def test_norm_writes_its_buffers_and_no_more(rows, width, dtype, buffers, cuda):
    lib, code, new = _native.library(), _native.dtype_code(dtype), normal(cuda, rows)
    x, w, b, grad = new(rows, width, dtype=dtype), new(width, dtype=dtype), new(width, dtype=dtype), new(rows, width, dtype=dtype)
    size, place = x.element_size(), (x.data_ptr(), rows, width, rows, 0, width)
    y, stats = buffers.new(rows * width * size), buffers.new(8 * rows)
    dx, dw, db = buffers.new(rows * width * size), buffers.new(width * size), buffers.new(width * size)
    room = lib.koemi_core_layer_norm_backward_workspace(rows, width)
    assert lib.koemi_core_layer_norm_forward(*place, w.data_ptr(), b.data_ptr(), code, y, stats, 1e-5, code, stream()) == 0
    assert lib.koemi_core_layer_norm_backward(*place, w.data_ptr(), code, stats, grad.data_ptr(), dx, dw, db, code, buffers.new(room), room, stream()) == 0
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    want = layer_norm(*leaves)
    for index, t in zip((0, 2, 3, 4), (want, *torch.autograd.grad(want, leaves, grad))):
        assert torch.equal(buffers.values(index, dtype, *t.shape), t)
    buffers.check()


@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("count", [1, 3, 7, 9, 4093, 1021 * 1021])
def test_dropout_writes_its_buffer_and_no_more(count, dtype, off, buffers, cuda):
    """Starts on and off 16 bytes, the last packet whole or not."""
    lib, x = _native.library(), normal(cuda, count)(count, dtype=dtype)
    for residual in (None, x):
        y = buffers.new(count * x.element_size(), off * x.element_size())
        assert lib.koemi_core_dropout(x.data_ptr(), None if residual is None else x.data_ptr(), y, count, 20000, 5, 6, 7, None, _native.dtype_code(dtype),
                                      stream()) == 0
        assert torch.equal(buffers.values(-1, dtype, count), dropout(x, 20000 / 65536, seed=5, site=6, step=7, residual=residual))
    buffers.check()


# ---------------------------------------------------------- streams at once

def test_training_passes_of_several_threads_on_streams_of_their_own(cuda):
    """Forward and backward of the whole sub-layer, sizes with different plans and workspaces in flight together; every
    result of every round has the bits of a call alone."""
    problems = []
    for k, (rows, width, hidden, dtype) in enumerate(((3, 64, 136, torch.bfloat16), (300, 512, 1024, torch.bfloat16), (4000, 96, 256, torch.float32),
                                                      (129, 200, 77, torch.float16), (9000, 64, 64, torch.bfloat16), (40, 16384, 40, torch.float32))):
        new = normal(cuda, k)
        leaves = [new(*s, scale=s[-1] ** -0.5, dtype=dtype) for s in ((hidden, width), (hidden, width), (width, hidden), (hidden,), (hidden,), (width,))]
        x, grad = new(rows, width, dtype=dtype), new(rows, width, dtype=dtype)
        problems.append(([t.requires_grad_(True) for t in (x, new(width), new(width), *leaves)], grad))

    def step(leaves, grad):
        x, nw, nb, wg, wv, wo, bg, bv, bo = leaves
        y = gated_feed_forward(layer_norm(x, nw, nb), wg, wv, wo, gate_bias=bg, value_bias=bv, output_bias=bo)
        y = dropout(y, 0.2, seed=3, residual=x)
        return (y.detach(), *torch.autograd.grad(y, leaves, grad))

    expected = [step(*problem) for problem in problems]
    ready = torch.cuda.Event()
    ready.record()
    errors, wrong = [], [torch.zeros((), dtype=torch.int64, device=cuda) for _ in problems]
    torch.cuda.synchronize()
    start = threading.Barrier(len(problems))

    def work(k):
        try:
            own = torch.cuda.Stream()
            own.wait_event(ready)
            with torch.cuda.stream(own):
                start.wait(60)
                for _ in range(40):
                    for got, want in zip(step(*problems[k]), expected[k]):
                        wrong[k].add_((got != want).sum())
            own.synchronize()
        except Exception as error:  # noqa: BLE001
            errors.append(error)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(len(problems))]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not errors, errors[0]
    assert [int(w) for w in wrong] == [0] * len(problems)


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


def test_batched_gradients_of_dropout(cuda):
    """A batch of gradients of one call: each has the call's mask."""
    new = normal(cuda)
    x, r, grads = new(40, 33).requires_grad_(True), new(40, 33).requires_grad_(True), new(5, 40, 33)
    y = dropout(x, 0.4, seed=2, site=1, step=torch.tensor(9, device=cuda), residual=r)
    dx, dr = torch.autograd.grad(y, (x, r), grads, is_grads_batched=True)
    assert torch.equal(dx, torch.stack([dropout(g, 0.4, seed=2, site=1, step=9) for g in grads])) and torch.equal(dr, grads)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_of_each_sample(dtype, cuda):
    """vmap of the norm's and the block's gradients: those of calls alone."""
    new = normal(cuda)
    x, nw = new(5, 40, 64, dtype=dtype), new(64, dtype=dtype)
    wg, wv, wo = new(48, 64, dtype=dtype), new(48, 64, dtype=dtype), new(64, 48, dtype=dtype)
    value = lambda t, nw, wg, wo: gated_feed_forward(layer_norm(t, nw), wg, wv, wo).float().square().sum()  # noqa: E731
    each = torch.func.grad(value, argnums=(0, 1, 2, 3))
    got = torch.vmap(each, in_dims=(0, None, None, None))(x, nw, wg, wo)
    for a, b in zip(got, zip(*(each(t, nw, wg, wo) for t in x))):
        assert torch.equal(a, torch.stack(b))
