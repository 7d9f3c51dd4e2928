"""The feed-forward sub-layer's operators called as training and serving programs call them: together, recomputed,
captured, on other streams, from several threads."""
from __future__ import annotations

import threading

import pytest
import torch
from torch.autograd import forward_ad
from torch.utils.checkpoint import checkpoint

from koemi_5hom_b200.cuda_kernels.core import dropout, layer_norm
from koemi_5hom_b200.cuda_kernels.dense import gated_feed_forward
from oracle import feed_forward as plain

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def parameters(width, hidden, dtype, cuda, seed=0):
    """Of the sub-layer: norm weight and bias, three weights, three biases."""
    g = torch.Generator().manual_seed(seed)
    normal = lambda scale, *shape: (scale * torch.randn(*shape, generator=g)).to(dtype).to(cuda).requires_grad_(True)  # noqa: E731
    norm = (1 + 0.1 * torch.randn(width, generator=g)).to(cuda).requires_grad_(True), (0.1 * torch.randn(width, generator=g)).to(cuda).requires_grad_(True)
    return [*norm, normal(width ** -0.5, hidden, width), normal(width ** -0.5, hidden, width), normal(hidden ** -0.5, width, hidden),
            normal(0.1, hidden), normal(0.1, hidden), normal(0.1, width)]


def sublayer(x, parameters, step=0, probability=0.1):
    nw, nb, wg, wv, wo, bg, bv, bo = parameters
    y = gated_feed_forward(layer_norm(x, nw, nb), wg, wv, wo, gate_bias=bg, value_bias=bv, output_bias=bo)
    return dropout(y, probability, seed=7, site=3, step=step, residual=x)


def plain_sublayer(x, parameters, step=0, probability=0.1):
    nw, nb, wg, wv, wo, bg, bv, bo = parameters
    y = plain.gated_feed_forward(plain.layer_norm(x, nw, nb), wg, wv, wo, bg, bv, bo)
    return plain.dropout(y, probability, 7, 3, step, x)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape,hidden", [((1, 1, 64), 128), ((3, 50, 96), 200), ((2, 700, 256), 512), ((4, 33, 515), 1030)], ids=str)
def test_the_sublayer_and_its_gradients(shape, hidden, dtype, cuda):
    """A whole step against 64 bits. No result goes through more than 12 roundings of the type, each of a root mean
    square of U / sqrt(3) of what it rounds and none grown by more than 2 on its way: 4 U of the result's norm. fp32
    rounds its sums, too: 32 instructions of a pass and some tens of terms' own, 2^-19."""
    g = torch.Generator().manual_seed(sum(shape))
    x, grad = (torch.randn(shape, generator=g).to(dtype).to(cuda) for _ in range(2))
    leaves = [x.requires_grad_(True), *parameters(shape[-1], hidden, dtype, cuda)]
    y = sublayer(leaves[0], leaves[1:])
    got = (y, *torch.autograd.grad(y, leaves, grad))
    exact = [t.detach().double().requires_grad_(True) for t in leaves]
    want = plain_sublayer(exact[0], exact[1:])
    want = (want, *torch.autograd.grad(want, exact, grad.double()))
    most = 4 * U[dtype] if dtype != torch.float32 else 2.0 ** -19
    for a, b in zip(got, want):
        assert a.shape == b.shape and (a.double() - b).norm().item() <= most * b.norm().item()
    with torch.no_grad():
        assert torch.equal(sublayer(x, leaves[1:]), y)


def test_a_batch_of_tokens_is_its_tokens(cuda):
    """Serving: a token's result does not depend on the batch, as far as its sums are cut alike: single tokens, whose
    K is cut finer, agree to the sums' roundings."""
    leaves = parameters(256, 512, torch.float32, cuda)
    x = torch.randn(64, 256, generator=torch.Generator().manual_seed(2)).to(cuda)
    with torch.no_grad():
        whole = sublayer(x, leaves, probability=0.0)
        single = torch.cat([sublayer(x[i:i + 1], leaves, probability=0.0) for i in range(64)])
    assert (whole - single).norm().item() <= 2.0 ** -19 * whole.norm().item()


def block_value(x):
    w = x[:40].reshape(-1)
    weights = w[:24 * 64].view(24, 64), w[100:100 + 24 * 64].view(24, 64), w[33:33 + 16 * 24].view(16, 24)
    return gated_feed_forward(x, *weights, gate_bias=w[:24], output_bias=w[50:66]).float().square().sum()


# an operator's scalar, and its input
VALUES = {"norm": (lambda x: layer_norm(x, x[0], x[1]).float().square().sum(), (300, 128), torch.bfloat16),
          "norm of wide rows": (lambda x: layer_norm(x, x[0].float(), None).square().sum(), (40, 16384), torch.float32),
          "norm of odd rows": (lambda x: layer_norm(x, x[0]).float().square().sum(), (200, 33), torch.float16),
          "dropout": (lambda x: dropout(x, 0.3, seed=1, residual=x * x).float().square().sum(), (300, 128), torch.bfloat16),
          "block": (block_value, (200, 64), torch.bfloat16), "block of fp32": (block_value, (200, 64), torch.float32),
          "block of a long sum": (block_value, (9000, 64), torch.bfloat16)}


@pytest.fixture(params=VALUES, ids=VALUES)
def operator(request, cuda):
    value, shape, dtype = VALUES[request.param]
    return value, torch.randn(shape, generator=torch.Generator().manual_seed(1)).to(dtype).to(cuda)


def gradient(value, x):
    leaf = x.detach().clone().requires_grad_(True)
    result = value(leaf)
    return result.detach(), torch.autograd.grad(result, leaf)[0]


def test_equal_calls_give_equal_bits(operator):
    value, x = operator
    first = gradient(value, x)
    for _ in range(10):
        assert all(torch.equal(a, b) for a, b in zip(first, gradient(value, x)))


def test_activation_checkpointing_gives_the_same_bits(operator):
    value, x = operator
    again = gradient(lambda t: checkpoint(value, t, use_reentrant=False), x)
    assert all(torch.equal(a, b) for a, b in zip(gradient(value, x), again))


def test_functional_gradients_give_the_same_bits(operator):
    value, x = operator
    assert torch.equal(torch.func.grad(value)(x), gradient(value, x)[1])


def test_forward_mode_is_refused(operator):
    value, x = operator
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        value(forward_ad.make_dual(x, torch.ones_like(x)))


def captured(call):
    """A graph of `call` after warm-up on a side stream, and what it returned."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        result = call()
    return graph, result


def test_forward_and_backward_in_cuda_graphs(operator):
    """Two graphs of the same call replayed in turn, on changed inputs."""
    value, x = operator
    x.requires_grad_(True)

    def call():
        result = value(x)
        return result, torch.autograd.grad(result, x)[0]

    graphs = [captured(call) for _ in range(2)]
    for turn in range(4):
        with torch.no_grad():
            x.copy_(x.roll(1, 0))
        graph, (result, grad) = graphs[turn % 2]
        graph.replay()
        expected = gradient(value, x)
        assert torch.equal(result, expected[0]) and torch.equal(grad, expected[1])


def test_on_another_stream(operator):
    value, x = operator
    expected = gradient(value, x)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        late = x.clone()
        for _ in range(50):  # still under way when the operator is launched
            late = late * 1
        got = gradient(value, late)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(expected, got))


def test_a_captured_training_step_draws_new_masks(cuda):
    """The program advances the step on the device; each replay has the masks of its step, forward and backward."""
    leaves = parameters(64, 128, torch.float32, cuda)
    x = torch.randn(90, 64, generator=torch.Generator().manual_seed(4)).to(cuda).requires_grad_(True)
    step = torch.zeros((), dtype=torch.int64, device=cuda)

    def call():
        y = sublayer(x, leaves, step=step, probability=0.5)
        grads = torch.autograd.grad(y, [x, *leaves], torch.ones_like(y))
        step.add_(1)
        return y, grads

    graph, (y, grads) = captured(call)
    step.fill_(100)
    for number in (100, 101, 102):
        graph.replay()
        with torch.enable_grad():
            expected = sublayer(x, leaves, step=number, probability=0.5)
            wanted = torch.autograd.grad(expected, [x, *leaves], torch.ones_like(expected))
        assert torch.equal(y, expected) and all(torch.equal(a, b) for a, b in zip(grads, wanted))


# calls of one kernel with different plans, workspaces and shared memory
SIZES = {"norm": (VALUES["norm"][0], [(300, 128), (20, 16384), (500, 33), (3, 40000)]),
         "block": (lambda x: gated_feed_forward(x, *(x[:1].expand(n, x.shape[1]) for n in (48, 48)), x[:1, :48].expand(8, 48)).float().sum(),
                   [(1, 64), (300, 2048), (4000, 96), (129, 200)]),
         "dropout": (VALUES["dropout"][0], [(1, 5), (300, 2048), (4000, 97)])}


@pytest.mark.parametrize("name", SIZES)
def test_threads_with_different_sizes(name, cuda):
    value, shapes = SIZES[name]
    inputs = [torch.randn(shape, generator=torch.Generator().manual_seed(3)).to(cuda).bfloat16() for shape in shapes]
    expected = [value(x) for x in inputs]
    errors = []

    def work(x, want):
        try:
            with torch.no_grad():
                for _ in range(300):
                    got = value(x)
                assert torch.equal(got, want)
        except Exception as error:  # noqa: BLE001
            errors.append(error)

    threads = [threading.Thread(target=work, args=pair) for pair in zip(inputs, expected)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not errors, errors[0]


def test_results_do_not_touch_what_lies_beside_them(cuda):
    """The C entries write their results and workspaces and no byte behind them."""
    from koemi_5hom_b200 import _native

    lib, stream = _native.library(), torch.cuda.current_stream().cuda_stream
    _native.ensure_device(cuda)
    for dtype, rows, width, hidden, out in ((torch.bfloat16, 3, 515, 77, 33), (torch.float32, 130, 40, 264, 65), (torch.float16, 257, 64, 128, 200)):
        code = _native.dtype_code(dtype)
        g = torch.Generator().manual_seed(rows)
        new = lambda *shape: (0.3 * torch.randn(*shape, generator=g)).to(dtype).to(cuda)  # noqa: E731
        guard = 1024

        def guarded(count, kind):
            buffer = torch.full((count * kind.itemsize + 2 * guard,), 0xA5, dtype=torch.uint8, device=cuda)
            return buffer, buffer.data_ptr() + guard

        x, wg, wv, wo, grad = new(rows, width), new(hidden, width), new(hidden, width), new(out, hidden), new(rows, out)
        sizes = [(rows * out, dtype), (lib.koemi_dense_gated_feed_forward_kept(rows, hidden, code), torch.uint8)]
        sizes += [(lib.koemi_dense_gated_feed_forward_workspace(rows, width, hidden, out, code, b), torch.uint8) for b in (0, 1)]
        sizes += [(n, dtype) for n in (rows * width, hidden * width, hidden * width, out * hidden, hidden, hidden, out)]
        buffers = [guarded(*size) for size in sizes]
        p = [b[1] for b in buffers]
        assert lib.koemi_dense_gated_feed_forward_forward(x.data_ptr(), width, wg.data_ptr(), wv.data_ptr(), wo.data_ptr(), None, None, None, p[0], p[1],
                                                          sizes[1][0], rows, width, hidden, out, code, p[2], sizes[2][0], stream) == 0
        assert lib.koemi_dense_gated_feed_forward_backward(x.data_ptr(), width, wg.data_ptr(), wv.data_ptr(), wo.data_ptr(), p[1], sizes[1][0],
                                                           grad.data_ptr(), *p[4:], rows, width, hidden, out, code, p[3], sizes[3][0], stream) == 0
        torch.cuda.synchronize()
        for (count, kind), (buffer, _) in zip(sizes, buffers):
            assert (buffer[:guard] == 0xA5).all() and (buffer[guard + count * kind.itemsize:] == 0xA5).all()
