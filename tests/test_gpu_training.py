"""Training operators on the GPU against plain 64-bit forms (oracle/training.py).

Tolerances. A result of type T is off by its own rounding, U[T] relative (half
a unit in the last place), plus what the fp32 arithmetic in front of it loses:
a count of roundings times 2^-24 (EPS) times the magnitude of the terms. Each
test derives its count where it uses it.
"""
from __future__ import annotations

import math
import threading

import pytest
import torch

from koemi_5hom_b200.cuda_kernels.core import clip_gradients, gradient_norm
from koemi_5hom_b200.cuda_kernels.dense import DenseCudaValidationError, gated_recurrence
from koemi_5hom_b200.cuda_kernels.moe import route_learned_topk
from koemi_5hom_b200.cuda_kernels.think import policy_loss
from oracle import training as plain

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}  # half the subnormal spacing
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def check(got, exact, dtype, absolute):
    """|got - exact| <= U |exact| + absolute, elementwise."""
    got, exact = got.double(), exact.double()
    allowed = U[dtype] * exact.abs() * 1.0001 + absolute + TINY[dtype]
    worst = ((got - exact).abs() - allowed).max().item() if got.numel() else -1.0
    assert got.shape == exact.shape and worst <= 0, f"off by {worst} more than allowed"


def normal(seed, *shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


# ------------------------------------------------------- the gated recurrence

def recurrence_case(batch, length, features, dtype, seed, masks, cuda, initial=True):
    g = torch.Generator().manual_seed(seed)
    x = (1.5 * torch.randn(batch, length, 2 * features, generator=g)).to(dtype).to(cuda)
    h0 = torch.randn(batch, features, generator=g).tanh().to(cuda) if initial else None
    valid = (torch.rand(batch, length, generator=g) < 0.8).to(cuda) if masks else None
    restart = (torch.rand(batch, length, generator=g) < 0.05).to(cuda) if masks else None
    gs = torch.randn(batch, length, features, generator=g).to(dtype).to(cuda)
    gf = torch.randn(batch, features, generator=g).to(cuda)
    return x, h0, valid, restart, gs, gf


def recurrence_bounds(x, h0):
    """Amplification 1 / (1 - max a) of a per-step error, and the largest state."""
    a = plain.LOW + (plain.HIGH - plain.LOW) * torch.sigmoid(x[..., :x.shape[-1] // 2].double())
    amplify = 1 / (1 - a.max().item()) if a.numel() else 1.0
    return min(amplify, max(1, x.shape[1])), max(1.0, h0.abs().max().item() if h0 is not None and h0.numel() else 1.0)


RECURRENCE_SHAPES = [(1, 1, 1), (3, 1, 64), (256, 1, 40), (2, 2, 33), (2, 8, 64), (3, 9, 16), (2, 63, 24), (1, 64, 128),
                     (2, 65, 8), (1, 129, 515), (3, 200, 64), (2, 511, 72), (1, 1025, 96), (5, 1000, 100), (1, 4097, 64),
                     (40, 130, 136)]


@pytest.mark.parametrize("masks", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", RECURRENCE_SHAPES)
def test_recurrence_and_gradients_match_the_plain_form(shape, dtype, masks, cuda):
    x, h0, valid, restart, gs, gf = recurrence_case(*shape, dtype, sum(shape), masks, cuda)
    states, final = gated_recurrence(x, h0, valid=valid, restart=restart)
    x64, h64 = x.double().requires_grad_(True), h0.double().requires_grad_(True)
    expected, expected_final = plain.gated_recurrence(x64, h64, valid, restart)
    # about ten roundings a step (sigmoid, tanh, the gate's and the state's products), each carried on with factor a
    amplify, most = recurrence_bounds(x, h0)
    lost = 16 * EPS * amplify * most
    assert states.dtype == dtype and final.dtype == torch.float32
    check(states, expected.detach(), dtype, lost)
    check(final, expected_final.detach(), torch.float32, lost)

    want_x, want_h = torch.autograd.grad((expected, expected_final), (x64, h64), (gs.double(), gf.double()))
    xg, hg = x.clone().requires_grad_(True), h0.clone().requires_grad_(True)
    states2, final2 = gated_recurrence(xg, hg, valid=valid, restart=restart)
    assert torch.equal(states2, states) and torch.equal(final2, final)
    got_x, got_h = torch.autograd.grad((states2, final2), (xg, hg), (gs, gf))
    # the adjoint sums |g| with weights a..., the state enters with its own loss
    adjoint = amplify * gs.abs().max().item() + gf.abs().max().item()
    check(got_x, want_x, dtype, 32 * EPS * amplify * adjoint * most)
    check(got_h, want_h, torch.float32, 16 * EPS * amplify * adjoint)


@pytest.mark.parametrize("masks", [False, True])
@pytest.mark.parametrize("shape", [(300, 130, 520), (320, 300, 264), (700, 20, 328)])
def test_recurrence_of_more_chains_than_the_gpu_holds(shape, masks, cuda):
    """Several chains walked by one CTA, one after the other."""
    x, h0, valid, restart, gs, gf = recurrence_case(*shape, torch.bfloat16, 17, masks, cuda)
    xg, hg = x.clone().requires_grad_(True), h0.clone().requires_grad_(True)
    states, final = gated_recurrence(xg, hg, valid=valid, restart=restart)
    got_x, got_h = torch.autograd.grad((states, final), (xg, hg), (gs, gf))
    amplify, most = recurrence_bounds(x, h0)
    adjoint = amplify * gs.abs().max().item() + gf.abs().max().item()
    for rows in (slice(0, 8), slice(shape[0] // 2, shape[0] // 2 + 8), slice(shape[0] - 8, shape[0])):
        x64, h64 = x[rows].double().requires_grad_(True), h0[rows].double().requires_grad_(True)
        expected, expected_final = plain.gated_recurrence(x64, h64, *(None if m is None else m[rows] for m in (valid, restart)))
        check(states[rows].detach(), expected.detach(), torch.bfloat16, 16 * EPS * amplify * most)
        check(final[rows].detach(), expected_final.detach(), torch.float32, 16 * EPS * amplify * most)
        want_x, want_h = torch.autograd.grad((expected, expected_final), (x64, h64), (gs[rows].double(), gf[rows].double()))
        check(got_x[rows], want_x, torch.bfloat16, 32 * EPS * amplify * adjoint * most)
        check(got_h[rows], want_h, torch.float32, 16 * EPS * amplify * adjoint)


@pytest.mark.parametrize("dtype", DTYPES)
def test_recurrence_carried_over_pieces_equals_one_call(dtype, cuda):
    x, h0, *_ = recurrence_case(2, 200, 48, dtype, 1, False, cuda)
    states, final = gated_recurrence(x, h0)
    h, pieces = h0, []
    for piece in x.split([1, 64, 70, 1, 64], 1):
        s, h = gated_recurrence(piece, h)
        pieces.append(s)
    amplify, most = recurrence_bounds(x, h0)
    check(torch.cat(pieces, 1), states.double(), dtype, 32 * EPS * amplify * most + U[dtype] * most)
    check(h, final.double(), torch.float32, 32 * EPS * amplify * most)


def test_recurrence_without_initial_and_with_one_gradient_only(cuda):
    x, _, valid, restart, gs, gf = recurrence_case(2, 150, 40, torch.float32, 2, True, cuda, initial=False)
    amplify, most = recurrence_bounds(x, None)
    for which, weight in ((0, gs), (1, gf)):
        xg, x64 = x.clone().requires_grad_(True), x.double().requires_grad_(True)
        got, = torch.autograd.grad(gated_recurrence(xg, valid=valid, restart=restart)[which], xg, weight)
        want, = torch.autograd.grad(plain.gated_recurrence(x64, None, valid, restart)[which], x64, weight.double())
        check(got, want, torch.float32, 32 * EPS * amplify * amplify * weight.abs().max().item() * most)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("length", [7, 300])
def test_recurrence_keeps_nan_out_of_masked_places(dtype, length, cuda):
    """NaN and infinities at positions that are not valid do nothing; those of one document end at a restart."""
    x, h0, valid, restart, gs, gf = recurrence_case(2, length, 64, dtype, 5, True, cuda)
    dirty = x.clone()
    dirty[~valid] = torch.tensor([math.nan, math.inf], device=cuda).repeat(64).to(dtype)
    a, b = x.clone().requires_grad_(True), dirty.requires_grad_(True)
    clean, soiled = (gated_recurrence(t, h0, valid=valid, restart=restart) for t in (a, b))
    assert torch.equal(clean[0], soiled[0]) and torch.equal(clean[1], soiled[1])
    grads = [torch.autograd.grad(out, t, (gs, gf))[0] for out, t in ((clean, a), (soiled, b))]
    assert torch.equal(*grads) and not grads[0][~valid].any()

    cut = length // 2
    bad = x.clone()
    bad[:, cut - 1] = math.nan
    edge = torch.zeros_like(valid)
    edge[:, cut] = True
    states, final = gated_recurrence(bad.requires_grad_(True), h0, restart=edge)
    after, last = gated_recurrence(x[:, cut:].contiguous())
    assert states[:, cut - 1].isnan().all() and not states[:, cut:].isnan().any()
    amplify, most = recurrence_bounds(x, h0)
    check(states[:, cut:].detach(), after.double(), dtype, 32 * EPS * amplify * most + U[dtype] * most)
    grad, = torch.autograd.grad((states, final), bad, (gs, gf))
    assert not grad[:, cut:].isnan().any()
    weights = torch.zeros_like(gs)
    weights[:, cut:] = math.nan  # nor does a NaN gradient cross the restart backwards
    states, final = gated_recurrence(a, h0, restart=edge)
    grad, = torch.autograd.grad(states, a, weights)
    assert not grad[:, :cut].any()


def test_recurrence_all_invalid_keeps_the_initial_state(cuda):
    x, h0, *_ = recurrence_case(2, 70, 24, torch.bfloat16, 6, False, cuda)
    h = h0.clone().requires_grad_(True)
    states, final = gated_recurrence(x, h, valid=torch.zeros(2, 70, dtype=torch.bool, device=cuda))
    assert torch.equal(final, h0) and torch.equal(states, h0.to(x.dtype).unsqueeze(1).expand_as(states))
    grad, = torch.autograd.grad(final, h, torch.ones_like(h0))
    assert torch.equal(grad, torch.ones_like(h0))


def test_recurrence_extreme_projections(cuda):
    """Saturated gates: a at its bounds, k at +-1, gradients zero or finite."""
    x = torch.tensor([0.0, 1e4, -1e4, 60.0, -60.0, 3e38, -3e38], device=cuda)
    x = torch.cartesian_prod(x, x).reshape(1, 49, 2).repeat(2, 2, 1)
    gx = x.clone().requires_grad_(True)
    states, final = gated_recurrence(gx)
    expected, _ = plain.gated_recurrence(x.cpu())
    check(states.detach().cpu(), expected, torch.float32, 16 * EPS * 256)
    grad, = torch.autograd.grad(states, gx, torch.ones_like(states))
    assert grad.isfinite().all()


def test_recurrence_empty_and_strided_inputs(cuda):
    x, h0, valid, restart, gs, _ = recurrence_case(3, 80, 32, torch.bfloat16, 8, True, cuda)
    states, final = gated_recurrence(x[:, :0], h0)
    assert states.shape == (3, 0, 32) and torch.equal(final, h0)
    assert gated_recurrence(x[:, :0])[1].eq(0).all()
    states, final = gated_recurrence(x[:0], h0[:0])
    assert states.shape == (0, 80, 32) and final.shape == (0, 32)
    wide = torch.cat((x, x), -1)
    expected = gated_recurrence(x, h0, valid=valid, restart=restart)
    got = gated_recurrence(wide[..., 64:], h0, valid=valid, restart=restart)
    turned = gated_recurrence(x.transpose(0, 1).contiguous().transpose(0, 1), h0.T.contiguous().T,
                              valid=valid.T.contiguous().T, restart=restart)
    for a, b, c in zip(expected, got, turned):
        assert torch.equal(a, b) and torch.equal(a, c)
    flat = torch.empty(x.numel() + 1, dtype=x.dtype, device=cuda)  # a base that no 16-byte load fits
    off = flat[1:].view_as(x).copy_(x)
    amplify, most = recurrence_bounds(x, h0)
    check(gated_recurrence(off, h0, valid=valid, restart=restart)[0], expected[0].double(), torch.bfloat16,
          32 * EPS * amplify * most + U[torch.bfloat16] * most)
    xg = off.clone().requires_grad_(True)
    out, _ = gated_recurrence(xg, h0, valid=valid, restart=restart)
    out.sum().backward()  # a gradient with strides of zero
    x64 = x.double().requires_grad_(True)
    want, = torch.autograd.grad(plain.gated_recurrence(x64, h0, valid, restart)[0].sum(), x64)
    check(xg.grad, want, torch.bfloat16, 32 * EPS * amplify * amplify * most)


def test_recurrence_gradient_by_differences(cuda):
    """Central differences along a direction: their own error is step^2 / 6 times
    a third derivative (of order 1 per element) and 2 * 16 EPS amplify sqrt(n) / (2 step)."""
    x, h0, valid, restart, gs, gf = recurrence_case(2, 130, 24, torch.float32, 11, True, cuda)
    v, vh = normal(12, *x.shape).to(cuda), normal(13, *h0.shape).to(cuda)

    def value(s):
        states, final = gated_recurrence(x + s * v, h0 + s * vh, valid=valid, restart=restart)
        return (states.double() * gs).sum().item() + (final.double() * gf).sum().item()

    xg, hg = x.clone().requires_grad_(True), h0.clone().requires_grad_(True)
    dx, dh = torch.autograd.grad(gated_recurrence(xg, hg, valid=valid, restart=restart), (xg, hg), (gs, gf))
    slope = (dx.double() * v).sum().item() + (dh.double() * vh).sum().item()
    step = 1e-2
    amplify, _ = recurrence_bounds(x, h0)
    n = math.sqrt(x.numel())
    assert abs((value(step) - value(-step)) / (2 * step) - slope) <= step ** 2 * n + 16 * EPS * amplify * n / step


@pytest.mark.parametrize("shape", [(1, 3000, 256), (64, 700, 64)])
def test_recurrence_bits_repeat_also_on_another_stream(shape, cuda):
    x, h0, valid, restart, gs, gf = recurrence_case(*shape, torch.bfloat16, 14, True, cuda)
    side, results = torch.cuda.Stream(), []
    for stream in (torch.cuda.current_stream(), side, side):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            xg, hg = x.clone().requires_grad_(True), h0.clone().requires_grad_(True)
            out = gated_recurrence(xg, hg, valid=valid, restart=restart)
            results.append([*out, *torch.autograd.grad(out, (xg, hg), (gs, gf))])
        torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))


def test_recurrence_as_a_threads_first_cuda_call(cuda):
    """A thread without a current context (an autograd thread is one) can encode tensor maps."""
    x, h0, *_ = recurrence_case(2, 100, 64, torch.bfloat16, 16, False, cuda)
    expected, got = gated_recurrence(x, h0), []
    thread = threading.Thread(target=lambda: got.extend(gated_recurrence(x, h0)))
    thread.start()
    thread.join()
    assert len(got) == 2 and all(torch.equal(a, b) for a, b in zip(got, expected))


def test_recurrence_offsets_past_32_bits(cuda):
    """2.2e9 projections: the last rows against the plain form from a carried state."""
    batch, length, features = 2, 8600, 64 * 1000
    x = torch.empty(batch, length, 2 * features, dtype=torch.bfloat16, device=cuda).normal_(generator=torch.Generator(cuda).manual_seed(3))
    restart = torch.zeros(batch, length, dtype=torch.bool, device=cuda)
    restart[:, -40] = True
    xg = x.requires_grad_(True)
    states, final = gated_recurrence(xg, restart=restart)
    tail = x[:, -40:].detach()
    expected, last = plain.gated_recurrence(tail)
    amplify, most = recurrence_bounds(tail, None)
    check(states[:, -40:].detach(), expected, torch.bfloat16, 16 * EPS * amplify * most)
    check(final.detach(), last, torch.float32, 16 * EPS * amplify * most)
    grad, = torch.autograd.grad(final, xg, torch.ones_like(final))
    t64 = tail.double().requires_grad_(True)
    want, = torch.autograd.grad(plain.gated_recurrence(t64)[1], t64, torch.ones_like(last))
    check(grad[:, -40:], want, torch.bfloat16, 32 * EPS * amplify * most)
    assert not grad[:, :-40].any()


def test_recurrence_in_a_cuda_graph(cuda):
    x, h0, *_ = recurrence_case(4, 1, 64, torch.bfloat16, 15, False, cuda)
    gated_recurrence(x, h0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = gated_recurrence(x, h0)
    x.copy_(torch.flip(x, [0]))
    graph.replay()
    expected = gated_recurrence(x, h0)
    assert all(torch.equal(a, b) for a, b in zip(captured, expected))


def test_recurrence_saved_tensors_are_guarded(cuda):
    """A changed input, a second backward of a freed graph and a second order are errors, not wrong gradients."""
    x, h0, *_ = recurrence_case(2, 40, 16, torch.float32, 18, False, cuda)
    y = x.clone().requires_grad_(True)
    z = y * 1.0
    states, _ = gated_recurrence(z, h0)
    states.sum().backward(retain_graph=True)
    first = y.grad.clone()
    y.grad = None
    states.sum().backward()
    assert torch.equal(first, y.grad)
    with pytest.raises(RuntimeError, match="second time"):
        states.sum().backward()
    z = y * 1.0
    states, _ = gated_recurrence(z, h0)
    with torch.no_grad():
        z.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        states.sum().backward()
    with pytest.raises(RuntimeError, match="first order"):
        torch.autograd.grad(gated_recurrence(y, h0)[0].sum(), y, create_graph=True)
    states, final = gated_recurrence(y, h0)
    states *= 2  # an output may be changed in place: nothing of it is kept
    got, = torch.autograd.grad(states.sum() + final.sum(), y)
    want, = torch.autograd.grad(2 * gated_recurrence(y, h0)[0].sum() + gated_recurrence(y, h0)[1].sum(), y)
    check(got, want.double(), torch.float32, 64 * EPS * 256)


def test_recurrence_of_turned_tensors_and_no_positions(cuda):
    """Strides are taken as they come, and gradients go back through them."""
    x, h0, *_ = recurrence_case(3, 37, 24, torch.float32, 19, False, cuda)
    turned, start = x.transpose(0, 1).contiguous().transpose(0, 1), h0.t().contiguous().t()
    grads = []
    for p, h in ((x, h0), (turned, start)):
        p, h = p.detach().requires_grad_(True), h.detach().requires_grad_(True)
        states, final = gated_recurrence(p, h)
        grads.append((states, *torch.autograd.grad(states.square().sum() + final.sum(), (p, h))))
    assert turned.stride() != x.stride() and all(torch.equal(a, b) for a, b in zip(*grads))
    p, h = x[:, :0].requires_grad_(True), h0.clone().requires_grad_(True)
    states, final = gated_recurrence(p, h)
    assert states.shape == (3, 0, 24) and torch.equal(final, h)
    final.sum().backward()
    assert torch.equal(h.grad, torch.ones_like(h))
    with pytest.raises(DenseCudaValidationError, match="initial must be float32"):
        gated_recurrence(p, h[:2])


def test_ops_refuse_what_the_kernels_cannot_take(cuda):
    """The dispatcher ops check for themselves, whoever calls them."""
    ops = torch.ops.koemi_b200
    x = torch.zeros(2, 5, 8, device=cuda)
    gated_recurrence(x)  # registers them
    carries, mask = torch.zeros(2, 1, 4, device=cuda), torch.ones(2, 5, dtype=torch.bool, device=cuda)
    logits, targets = torch.zeros(6, 9, device=cuda), torch.zeros(6, dtype=torch.int64, device=cuda)
    rows, one = torch.zeros(6, device=cuda), torch.ones((), device=cuda)
    pairs, ids = torch.zeros(6, 2, device=cuda), torch.zeros(6, 2, dtype=torch.int64, device=cuda)
    for call in (lambda: ops.gated_recurrence(x, None, mask[:, :4], None, 0.1, 0.9),
                 lambda: ops.gated_recurrence(x, None, None, mask[:1], 0.1, 0.9),
                 lambda: ops.gated_recurrence(x, carries[:, 0, :3], None, None, 0.1, 0.9),
                 lambda: ops.gated_recurrence(x, None, None, None, 0.9, 0.1),
                 lambda: ops.gated_recurrence(x.cpu(), carries[:, 0], None, None, 0.1, 0.9),
                 lambda: ops.gated_recurrence_keep(x.transpose(0, 1), None, None, None, 0.1, 0.9),
                 lambda: ops.gated_recurrence_keep(x[:, :0], None, None, None, 0.1, 0.9),
                 lambda: ops.gated_recurrence_backward(x, None, None, carries[:, :0], None, None, 0.1, 0.9),
                 lambda: ops.gated_recurrence_backward(x, None, None, carries, x, None, 0.1, 0.9),
                 lambda: ops.route_learned(logits, None, 10, False),
                 lambda: ops.route_learned(logits, mask[0], 1, False),
                 lambda: ops.route_learned_backward(logits, ids, pairs[:5], rows[:5], None, None, False),
                 lambda: ops.route_learned_backward(logits, ids, pairs, rows, None, None, False),
                 lambda: ops.policy_loss(logits, targets[:5], rows, rows, None, None, 0.2, 0.2, 0.0),
                 lambda: ops.policy_loss(logits, targets, rows[:5], rows, None, None, 0.2, 0.2, 0.0),
                 lambda: ops.policy_loss(logits, targets, rows, rows, None, None, 0.2, 0.2, 1.0),
                 lambda: ops.policy_loss(logits, targets, rows, rows, rows.double(), None, 0.2, 0.2, 0.0),
                 lambda: ops.policy_loss(logits, targets, rows, rows, None, None, -0.2, 0.2, 0.0),
                 lambda: ops.policy_loss_backward(logits, targets, None, pairs, one),
                 lambda: ops.policy_loss_scale(logits, rows)):
        with pytest.raises(ValueError):
            call()


# ------------------------------------------------------------ the learned route

def route_case(tokens, experts, top_k, dtype, seed, masks, cuda):
    g = torch.Generator().manual_seed(seed)
    x = (1.5 * torch.randn(tokens, experts, generator=g)).to(dtype).to(cuda)
    valid = (torch.rand(tokens, generator=g) < 0.8).to(cuda) if masks else None
    return x, valid, torch.randn(tokens, top_k, generator=g).to(cuda)


ROUTE_SHAPES = [(1, 1, 1), (1, 64, 2), (256, 64, 2), (7, 3, 3), (33, 128, 8), (1000, 17, 4), (1000, 33, 1), (777, 122, 5),
                (300, 257, 2), (90, 1000, 16), (5, 4096, 256), (20000, 8, 2)]


@pytest.mark.parametrize("masks,renormalize", [(False, False), (True, True), (True, False), (False, True)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", ROUTE_SHAPES)
def test_route_and_gradients_match_the_plain_form(shape, dtype, masks, renormalize, cuda):
    tokens, experts, top_k = shape
    x, valid, gw = route_case(*shape, dtype, sum(shape), masks, cuda)
    gb = torch.tensor(0.7, device=cuda)
    xg, x64 = x.clone().requires_grad_(True), x.double().requires_grad_(True)
    route = route_learned_topk(xg, valid, top_k=top_k, renormalize=renormalize)
    ids, weights, counts, balance = plain.route_learned(x64, valid, top_k, renormalize)
    assert torch.equal(route.expert_ids, ids) and torch.equal(route.counts, counts)
    # exp loses |l - max| roundings (at most 16 here), its sum 32 + log2(E), the products a few
    lost = 64 * EPS
    check(route.weights.detach(), weights.detach(), torch.float32, lost)
    check(route.balance_loss.detach(), balance.detach(), torch.float32, lost * max(1.0, balance.item()))
    got, = torch.autograd.grad((route.weights, route.balance_loss), xg, (gw, gb))
    want, = torch.autograd.grad((weights, balance), x64, (gw.double(), gb.double()))
    total = torch.softmax(x.double(), -1).gather(-1, ids.clamp_min(0)).sum(-1).min().item() if renormalize else 1.0
    assert got.dtype == dtype
    check(got, want, dtype, 4 * lost * (gw.abs().max().item() / total + 0.7 * experts / tokens))
    inference = route_learned_topk(x, valid, top_k=top_k, renormalize=renormalize)
    assert torch.equal(inference.expert_ids, route.expert_ids) and torch.equal(inference.weights, route.weights.detach())


def test_route_ties_go_to_the_lowest_expert(cuda):
    x = torch.zeros(4, 40, device=cuda)
    x[1, 5:] = 1.0
    x[2, ::2] = -math.inf
    x[3] = torch.finfo(torch.float32).min
    ids = route_learned_topk(x, top_k=3).expert_ids.tolist()
    assert ids == [[0, 1, 2], [5, 6, 7], [1, 3, 5], [0, 1, 2]]


@pytest.mark.parametrize("experts", [4, 64, 300])
def test_route_masked_experts_and_rows_that_leave_nothing(experts, cuda):
    x = normal(3, 6, experts).to(cuda)
    x[0] = -math.inf                       # nothing left
    x[1, 1:] = -math.inf                   # one expert left, two wanted
    x[2, :2] = torch.finfo(torch.float32).min
    x[3] = math.nan                        # not valid: never looked at
    x[4] = math.inf
    valid = torch.tensor([True, True, True, False, False, True], device=cuda)
    xg = x.clone().requires_grad_(True)
    route = route_learned_topk(xg, valid, top_k=2, renormalize=True)
    x64 = x.double().requires_grad_(True)
    ids, weights, counts, balance = plain.route_learned(x64, valid, 2, True)
    assert torch.equal(route.expert_ids, ids) and torch.equal(route.counts, counts)
    assert route.expert_ids[0].tolist() == [-1, -1] and route.expert_ids[1].tolist() == [0, 1]
    assert route.counts.sum().item() == 6
    check(route.weights.detach(), weights.detach(), torch.float32, 64 * EPS)
    check(route.balance_loss.detach(), balance.detach(), torch.float32, 64 * EPS * experts)
    grad, = torch.autograd.grad((route.weights.sum(), route.balance_loss), xg)
    assert not grad[[0, 3, 4]].any() and grad.isfinite().all()


def test_route_without_a_live_row_and_without_rows(cuda):
    x = normal(4, 5, 8).to(cuda).requires_grad_(True)
    route = route_learned_topk(x, torch.zeros(5, dtype=torch.bool, device=cuda), top_k=2)
    assert route.balance_loss.item() == 0 and not route.counts.any() and (route.expert_ids == -1).all()
    grad, = torch.autograd.grad((route.weights.sum(), route.balance_loss), x)
    assert not grad.any()
    route = route_learned_topk(torch.zeros(0, 8, device=cuda), top_k=2)
    assert route.balance_loss.item() == 0 and not route.counts.any() and route.expert_ids.shape == (0, 2)


def test_route_nan_logits_are_never_preferred(cuda):
    x = normal(5, 3, 50).to(cuda)
    x[1, 7] = math.nan
    route = route_learned_topk(x, top_k=4)
    assert 7 not in route.expert_ids[1].tolist() and route.weights[1].isnan().all()
    assert not route.weights[[0, 2]].isnan().any()
    x[1] = math.nan
    assert route_learned_topk(x, top_k=4).expert_ids[1].tolist() == [0, 1, 2, 3]


def test_route_one_gradient_only_and_strided_logits(cuda):
    wide = normal(6, 100, 96).to(cuda)
    x = wide[:, 8:72]
    for which in (0, 1):
        xg, x64 = x.clone().requires_grad_(True), x.double().requires_grad_(True)
        r, p = route_learned_topk(xg, top_k=2), plain.route_learned(x64, None, 2, False)
        got, = torch.autograd.grad((r.weights, r.balance_loss)[which].sum(), xg)
        want, = torch.autograd.grad((p[1], p[3])[which].sum(), x64)
        check(got, want, torch.float32, 256 * EPS)
    a, b = route_learned_topk(x, top_k=2), route_learned_topk(x.contiguous(), top_k=2)
    assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_route_gradient_by_differences(cuda):
    """Differences of the weights and the loss along a direction that changes no
    choice: step^2 times third derivatives of order 1, and 64 EPS sqrt(n) / step."""
    x = (torch.argsort(normal(7, 64, 24), -1).float() * 0.1).to(cuda)  # logits 0.1 apart
    v = normal(8, 64, 24).clamp(-2, 2).to(cuda)
    gw = normal(9, 64, 3).to(cuda)

    def value(s):
        r = route_learned_topk(x + s * v, top_k=3, renormalize=True)
        return (r.weights.double() * gw).sum().item() + 5 * r.balance_loss.double().item()

    xg = x.clone().requires_grad_(True)
    r = route_learned_topk(xg, top_k=3, renormalize=True)
    grad, = torch.autograd.grad((r.weights, r.balance_loss), xg, (gw, torch.tensor(5.0, device=cuda)))
    step = 1e-2
    n = math.sqrt(x.numel())
    assert abs((value(step) - value(-step)) / (2 * step) - (grad.double() * v).sum().item()) <= step ** 2 * n + 64 * EPS * n / step


def test_route_bits_repeat(cuda):
    x, valid, gw = route_case(30000, 64, 2, torch.float32, 10, True, cuda)
    first = route_learned_topk(x, valid, top_k=2)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, route_learned_topk(x, valid, top_k=2)))


# ------------------------------------------------------------- the policy loss

def policy_case(rows, vocab, dtype, seed, cuda, shape=None):
    g = torch.Generator().manual_seed(seed)
    logits = (2.5 * torch.randn(rows, vocab, generator=g)).to(dtype)
    targets = torch.randint(0, vocab, (rows,), generator=g)
    lp = torch.log_softmax(logits.double(), -1).gather(-1, targets[:, None])[:, 0]
    drift = 0.2 * torch.randn(rows, generator=g).double()
    for edge in (math.log(0.8), math.log(1.3)):  # a ratio on an edge has no unique gradient
        drift = torch.where((drift - edge).abs() < 1e-3, edge + 2e-3, drift)
    case = dict(logits=logits, targets=targets, old=(lp - drift).float(), advantages=torch.randn(rows, generator=g),
                reference=(lp + 0.1 * torch.randn(rows, generator=g)).float(), valid=torch.rand(rows, generator=g) < 0.8)
    case["valid"][0] = True
    shape = shape or (rows,)
    return {k: (t.reshape(*shape, vocab) if k == "logits" else t.reshape(shape)).to(cuda) for k, t in case.items()}


def run_policy(case, valid=True, reference=True, scale=None, logits=None):
    logits = case["logits"].detach().clone().requires_grad_(True) if logits is None else logits
    result = policy_loss(logits, case["targets"], case["old"], case["advantages"],
                         reference_log_probs=case["reference"] if reference else None,
                         valid_mask=case["valid"] if valid else None, clip_low=0.2, clip_high=0.3,
                         kl_weight=0.05 if reference else 0.0)
    grad, = torch.autograd.grad(result.loss, logits, None if scale is None else torch.tensor(scale, device=logits.device))
    return result, grad


def plain_policy(case, valid=True, reference=True, scale=1.0):
    x = case["logits"].double().requires_grad_(True)
    loss, kl, lp = plain.policy_loss(x, case["targets"], case["old"], case["advantages"], case["reference"] if reference else None,
                                     case["valid"] if valid else None, 0.2, 0.3, 0.05)
    return loss.detach(), kl.detach(), lp.detach(), torch.autograd.grad(loss, x, torch.tensor(scale, dtype=torch.float64, device=x.device))[0]


def check_policy(case, result, grad, expected, scale=1.0):
    loss, kl, lp, want = expected
    dtype = case["logits"].dtype
    rows = case["targets"].numel()
    # the log-sum-exp: |l - max| roundings in the exponentials (up to 32), about 40 in the sum, then two roundings at
    # its own magnitude (up to 32); a ratio inherits that, times |A|, and the KL term, times e^d
    lost = (32 + 40 + 2 * 32) * EPS
    ratio = torch.where(case["valid"], torch.exp(lp - case["old"]), 0.0).max().item()
    gap = torch.where(case["valid"], torch.exp(case["reference"] - lp), 0.0).max().item()
    size = max(3.0, ratio, gap) * max(1.0, case["advantages"].abs().max().item())
    check(result.log_probs, lp, torch.float32, lost)
    check(result.loss.detach(), loss, torch.float32, lost * size)
    check(result.kl, kl, torch.float32, lost * max(1.0, gap))
    count = max(1, int(case["valid"].sum()))
    rounds = 1 if scale == 1.0 else 2  # written once, scaled once
    check(grad, want, dtype, scale * lost * size / count + (rounds - 1) * U[dtype] * want.abs().max().item())
    assert grad.dtype == dtype and grad.shape == case["logits"].shape and rows == result.log_probs.numel()


POLICY_SHAPES = [(1, 1), (3, 2), (5, 31), (64, 257), (33, 256), (9, 1000), (17, 1024), (10, 4097), (7, 8200), (700, 320),
                 (5, 32767), (6, 32768), (3, 65000), (2, 131072), (2, 250001)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", POLICY_SHAPES)
def test_policy_loss_and_gradient_match_the_plain_form(shape, dtype, cuda):
    case = policy_case(*shape, dtype, sum(shape), cuda)
    scale = 64.0 if dtype == torch.float16 else None
    result, grad = run_policy(case, scale=scale)
    check_policy(case, result, grad, plain_policy(case, scale=scale or 1.0), scale or 1.0)
    assert not grad[~case["valid"]].any() and not result.log_probs[~case["valid"]].any()
    evaluated = policy_loss(case["logits"], case["targets"], case["old"], case["advantages"], reference_log_probs=case["reference"],
                            valid_mask=case["valid"], clip_low=0.2, clip_high=0.3, kl_weight=0.05)
    assert torch.equal(evaluated.loss, result.loss) and torch.equal(evaluated.log_probs, result.log_probs)


@pytest.mark.parametrize("dtype", DTYPES)
def test_policy_loss_of_strided_logits(dtype, cuda):
    """All positions but the last, as next-token losses take them, a slice of the vocabulary, and a transposed batch."""
    whole = policy_case(4 * 9, 264, dtype, 3, cuda, shape=(4, 9))
    views = {"positions": lambda t: t[:, :-1], "turned": lambda t: t.transpose(0, 1)}
    for name, view in views.items():
        case = {k: view(t) for k, t in whole.items()}
        scale = 64.0 if dtype == torch.float16 else None
        leaf = whole["logits"].clone().requires_grad_(True)
        result, grad = run_policy(case, scale=scale, logits=view(leaf))
        check_policy(case, result, grad, plain_policy(case, scale=scale or 1.0), scale or 1.0)
    case = dict(whole, logits=whole["logits"][..., 3:260], targets=whole["targets"] % 257)
    result, grad = run_policy(case, logits=whole["logits"].clone().requires_grad_(True)[..., 3:260], scale=64.0)
    check_policy(case, result, grad, plain_policy(case, scale=64.0), 64.0)


@pytest.mark.parametrize("valid,reference", [(False, True), (True, False), (False, False)])
def test_policy_loss_without_mask_or_reference(valid, reference, cuda):
    case = policy_case(50, 300, torch.float32, 4, cuda)
    if not valid:
        case["valid"] = torch.ones_like(case["valid"])
    result, grad = run_policy(case, valid, reference)
    check_policy(case, result, grad, plain_policy(case, valid, reference))


@pytest.mark.parametrize("vocab", [257, 4096, 40000])
def test_policy_masked_rows_are_not_read(vocab, cuda):
    case = policy_case(12, vocab, torch.bfloat16, 5, cuda)
    result, grad = run_policy(case)
    dirty = dict(case, logits=case["logits"].clone(), targets=case["targets"].clone(), old=case["old"].clone())
    out = ~case["valid"]
    dirty["logits"][out], dirty["old"][out], dirty["targets"][out] = math.nan, math.inf, -5
    again, grad2 = run_policy(dirty)
    assert torch.equal(result.loss, again.loss) and torch.equal(grad, grad2) and torch.equal(result.log_probs, again.log_probs)
    case["valid"] = torch.zeros_like(case["valid"])
    result, grad = run_policy(case)
    assert result.loss.item() == 0 and result.kl.item() == 0 and not grad.any()


@pytest.mark.parametrize("vocab", [257, 4096, 40000])
@pytest.mark.parametrize("low", [-math.inf, torch.finfo(torch.float32).min])
def test_policy_masked_vocabulary(vocab, low, cuda):
    """Forbidden tokens at -inf or the type's lowest value: probability and gradient zero."""
    case = policy_case(8, vocab, torch.float32, 6, cuda)
    forbidden = torch.zeros(8, vocab, dtype=torch.bool, device=cuda)
    forbidden[:, ::3] = True
    forbidden.scatter_(1, case["targets"][:, None], False)
    case["logits"] = torch.where(forbidden, low, case["logits"])
    result, grad = run_policy(case)
    expected = plain_policy(case)
    size = 3 * 8 * case["advantages"].abs().max().item()
    ratio = torch.exp(expected[2] - case["old"]).max().item()  # the ratios are no longer near one
    check(result.log_probs, expected[2], torch.float32, 136 * EPS)
    check(grad, expected[3].nan_to_num(0.0), torch.float32, 136 * EPS * size * max(1.0, ratio))
    assert not grad[forbidden].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [900, 8000, 32768, 70000])
def test_policy_masked_halves_beside_very_low_logits(vocab, dtype, cuda):
    """A run of forbidden entries longer than any thread's or warp's share, beside logits near -200: e^200 must not
    meet their zeros."""
    case = policy_case(4, vocab, dtype, 16, cuda)
    half = vocab // 2
    case["targets"] %= half
    case["logits"] = (case["logits"].float() - 200).to(dtype)
    case["logits"][:, half:] = -math.inf
    case["logits"][3] = torch.finfo(dtype).min  # a row of the type's lowest value: uniform
    lp = torch.log_softmax(case["logits"].double(), -1).gather(-1, case["targets"][:, None])[:, 0]
    case["old"], case["reference"] = (lp - 0.1).float(), (lp + 0.1).float()
    scale = 64.0 if dtype == torch.float16 else None
    result, grad = run_policy(case, scale=scale)
    # a log-sum-exp near -200 rounds at 16 times the magnitude of the ones above; the uniform row's at the lowest value's
    check(result.log_probs[:3], plain_policy(case)[2][:3], torch.float32, (32 + 40 + 2 * 256) * EPS)
    assert grad.isfinite().all() and not grad[:3, half:].any()
    size = 3 * max(1.0, case["advantages"].abs().max().item()) * (scale or 1.0)
    rounds = (1 if scale is None else 2) * U[dtype]
    want = plain_policy(case, scale=scale or 1.0)[3]
    check(grad[:3], want[:3], dtype, 2 * (32 + 40 + 2 * 256) * EPS * size + rounds * want[:3].abs().max().item())


def test_policy_bad_targets_are_loud_and_local(cuda):
    case = policy_case(6, 500, torch.float32, 7, cuda)
    case["valid"][:] = True
    case["targets"][2], case["targets"][4] = 500, -1
    result, grad = run_policy(case)
    bad = torch.tensor([2, 4], device=cuda)
    assert result.loss.isnan() and result.log_probs[bad].isnan().all() and grad[bad].isnan().all()
    good = torch.tensor([0, 1, 3, 5], device=cuda)
    assert not result.log_probs[good].isnan().any() and not grad[good].isnan().any()


def test_policy_second_backward_and_in_place_loss(cuda):
    case = policy_case(20, 700, torch.bfloat16, 8, cuda)
    logits = case["logits"].requires_grad_(True)
    result = policy_loss(logits, case["targets"], case["old"], case["advantages"], valid_mask=case["valid"])
    first, = torch.autograd.grad(result.loss, logits, torch.tensor(3.0, device=cuda), retain_graph=True)
    second, = torch.autograd.grad(result.loss, logits, torch.tensor(3.0, device=cuda))
    largest = first.abs().max().item()
    check(first, second.double(), torch.bfloat16, U[torch.bfloat16] * largest * 2)
    loss = policy_loss(logits, case["targets"], case["old"], case["advantages"], valid_mask=case["valid"]).loss
    loss /= 4
    loss.backward()
    check(logits.grad, second.double() / 12, torch.bfloat16, U[torch.bfloat16] * largest)


def test_policy_gradient_by_differences(cuda):
    """step^2 times third derivatives (ratios, softmax: below 4 |A| a row) and 136 EPS |A| / step."""
    case = policy_case(16, 300, torch.float32, 9, cuda)
    v = normal(10, 16, 300).to(cuda)
    _, grad = run_policy(case)

    def value(s):
        return policy_loss(case["logits"] + s * v, case["targets"], case["old"], case["advantages"],
                           reference_log_probs=case["reference"], valid_mask=case["valid"], clip_low=0.2, clip_high=0.3,
                           kl_weight=0.05).loss.double().item()

    step = 2e-4  # the ratios stay 1e-3 from the edges, a log-prob moves by at most about 4 steps
    size = case["advantages"].abs().max().item()
    assert abs((value(step) - value(-step)) / (2 * step) - (grad.double() * v).sum().item()) <= 4 * size * step ** 2 * 64 + 136 * EPS * size / step


def test_policy_bits_repeat(cuda):
    case = policy_case(900, 515, torch.bfloat16, 12, cuda)
    first, grad = run_policy(case)
    for _ in range(3):
        again, grad2 = run_policy(case)
        assert torch.equal(first.loss, again.loss) and torch.equal(first.kl, again.kl) and torch.equal(grad, grad2)


@pytest.mark.parametrize("vocab,dtype", [(1030, torch.float32), (4097, torch.bfloat16), (16397, torch.float16),
                                         (33001, torch.float32), (70003, torch.bfloat16)])
def test_policy_ragged_rows_at_the_ends_of_their_storage(vocab, dtype, cuda):
    """Rows of odd lengths that start one element into a storage and end with it, between NaN where it has room."""
    rows = 7
    case = policy_case(rows, vocab, dtype, vocab, cuda)
    scale = 64.0 if dtype == torch.float16 else None
    expected = plain_policy(case, scale=scale or 1.0)
    for stride in (vocab, vocab + 3):
        storage = torch.full((1 + (rows - 1) * stride + vocab,), math.nan, dtype=dtype, device=cuda)
        logits = storage.as_strided((rows, vocab), (stride, 1), 1)
        logits.copy_(case["logits"])
        result, grad = run_policy(case, scale=scale, logits=logits.detach().requires_grad_(True))
        check_policy(case, result, grad, expected, scale or 1.0)


def test_policy_many_rows_of_a_cta(cuda):
    """512 times the same 40 rows: more than a CTA's table of row scalars holds."""
    case = policy_case(40, 16400, torch.bfloat16, 21, cuda)
    loss, kl, lp, want = plain_policy(case)
    many = {k: t.repeat(512, *[1] * (t.ndim - 1)) for k, t in case.items()}
    result, grad = run_policy(many)
    size = 136 * EPS * 3 * max(1.0, case["advantages"].abs().max().item())
    check(result.loss.detach(), loss, torch.float32, size)
    check(result.kl, kl, torch.float32, size)
    check(result.log_probs, lp.repeat(512), torch.float32, 136 * EPS)
    assert torch.equal(grad.view(512, 40, -1), grad[:40].expand(512, -1, -1))  # equal rows, equal bits
    count = int(case["valid"].sum())
    check(grad[:40] * 512, want, torch.bfloat16, size / count)


def test_policy_offsets_past_32_bits(cuda):
    """70000 rows of 32768: only the last ones are valid."""
    rows, vocab = 70000, 32768
    tail = policy_case(5, vocab, torch.bfloat16, 13, cuda)
    tail["valid"][:] = True
    logits = torch.zeros(rows, vocab, dtype=torch.bfloat16, device=cuda)
    logits[-5:] = tail["logits"]
    case = {"logits": logits}
    for k in ("targets", "old", "advantages", "reference", "valid"):
        case[k] = torch.zeros(rows, dtype=tail[k].dtype, device=cuda)
        case[k][-5:] = tail[k]
    result, grad = run_policy(case, logits=logits.requires_grad_(True))
    loss, kl, lp, want = plain_policy(tail)
    check(result.log_probs[-5:], lp, torch.float32, 136 * EPS)
    check(grad[-5:], want, torch.bfloat16, 136 * EPS * 10)
    assert not grad[:-5].any()


# ------------------------------------------------------ the clipping of gradients

def gradient_list(shapes, dtypes, seed, cuda, scale=0.1):
    return [(scale * normal(seed + i, *s)).to(dtypes[i % len(dtypes)]).to(cuda) for i, s in enumerate(shapes)]


# squares are added up in runs of at most 64, then over 8 warps of 32 lanes; the root halves the loss
NORM_LOST = 128 * EPS
CLIP_SHAPES = [[(1,)], [(5,), (0,), (3, 7), ()], [(16384,), (16385,), (16383,), (1,)], [(100, 333), (64, 64), (7,), (40001,)],
               [(300000,)], [(3,)] * 1500, [(1 << 21,), ((1 << 21) + 1,)]]


@pytest.mark.parametrize("dtypes", [[torch.float32], [torch.bfloat16], [torch.float16], [torch.bfloat16, torch.float32, torch.float16]])
@pytest.mark.parametrize("shapes", CLIP_SHAPES, ids=lambda s: f"{len(s)}x{s[0]}")
@pytest.mark.parametrize("max_norm", [1.0, 1e4])
def test_clip_matches_the_plain_form(shapes, dtypes, max_norm, cuda):
    gradients = gradient_list(shapes, dtypes, 1, cuda)
    norm, expected = plain.clip_gradients(gradients, max_norm)
    kept = [g.clone() for g in gradients]
    out = [torch.full_like(g, math.nan) for g in gradients]
    got = clip_gradients(gradients, max_norm, out=out)
    assert got.dtype == torch.float32 and got.shape == ()
    check(got, norm, torch.float32, NORM_LOST * norm.item())
    for o, e, g, k in zip(out, expected, gradients, kept):
        check(o, e, o.dtype, NORM_LOST * (e.abs().max().item() if e.numel() else 0.0))
        assert torch.equal(g, k)
    assert torch.equal(gradient_norm(gradients), got)
    assert torch.equal(clip_gradients(gradients, max_norm), got)
    assert all(torch.equal(g, o) for g, o in zip(gradients, out))


@pytest.mark.parametrize("dtype", DTYPES)
def test_clip_of_views_into_flat_buffers(dtype, cuda):
    """Neighbours at every alignment, outputs aligned as the gradients and otherwise."""
    sizes = [1, 2, 3, 5, 4099, 8, 16390, 7, 33000, 12, 1]
    flat = normal(2, sum(sizes)).to(dtype).to(cuda)
    gradients = list(flat.split(sizes))
    norm, expected = plain.clip_gradients(gradients, 2.0)
    for shift in (0, 1, 3):
        room = torch.full((sum(sizes) + 8,), 7.0, dtype=dtype, device=cuda)
        out = list(room[shift:shift + sum(sizes)].split(sizes))
        check(clip_gradients(gradients, 2.0, out=out), norm, torch.float32, NORM_LOST * norm.item())
        for o, e in zip(out, expected):
            check(o, e, dtype, NORM_LOST * e.abs().max().item())
        assert (room[:shift] == 7).all() and (room[shift + sum(sizes):] == 7).all()


def test_clip_leaves_small_gradients_alone_and_is_stable(cuda):
    gradients = gradient_list([(1000,), (77,)], [torch.bfloat16], 3, cuda)
    kept = [g.clone() for g in gradients]
    norm = clip_gradients(gradients, math.inf)
    assert all(torch.equal(g, k) for g, k in zip(gradients, kept))
    for _ in range(3):
        assert torch.equal(clip_gradients(gradients, 1e9), norm)
    out = [torch.zeros_like(g) for g in gradients]
    clip_gradients(gradients, 1e9, out=out)
    assert all(torch.equal(g, o) for g, o in zip(gradients, out))
    clip_gradients(gradients, 0.0)
    assert not any(g.any() for g in gradients)
    assert clip_gradients(gradients, 1.0).item() == 0.0 and not any(g.any() for g in gradients)


def test_clip_of_infinite_and_nan_gradients(cuda):
    gradients = gradient_list([(100,), (50,)], [torch.float32], 4, cuda)
    gradients[0][3] = math.inf
    out = [torch.zeros_like(g) for g in gradients]
    assert clip_gradients(gradients, 1.0, out=out).item() == math.inf
    assert out[0][3].isnan() and not out[0][:3].any() and not out[1].any()
    gradients[1][2] = math.nan
    assert clip_gradients(gradients, 1.0, out=out).isnan() and all(o.isnan().all() for o in out)


def test_clip_of_one_tensor_past_32_bits(cuda):
    flat = torch.zeros((1 << 31) + 100, dtype=torch.bfloat16, device=cuda)
    flat[5], flat[-1], flat[1 << 31] = 3.0, 4.0, 12.0
    assert clip_gradients([flat], 6.5).item() == 13.0
    # 6.5 / (13 + 1e-6) rounds to just below one half, the products to the same bf16 as exact halves
    assert flat[5].item() == 1.5 and flat[-1].item() == 2.0 and flat[1 << 31].item() == 6.0


def test_clip_matches_an_optimizer_step_in_a_graph(cuda):
    gradients = gradient_list([(64, 64), (64,)], [torch.float32], 6, cuda)
    clip_gradients(gradients, 1.0, out=[g.clone() for g in gradients])
    out = [torch.zeros_like(g) for g in gradients]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_gradients(gradients, 1.0, out=out)
    for g in gradients:
        g.mul_(2.0)
    graph.replay()
    expected, clipped = plain.clip_gradients(gradients, 1.0)
    check(norm, expected, torch.float32, NORM_LOST * expected.item())
    for o, e in zip(out, clipped):
        check(o, e, torch.float32, NORM_LOST * e.abs().max().item())
