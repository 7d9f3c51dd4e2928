"""The training operators' results entry by entry against 64-bit forms, with bounds carried through the formulas.

A result of type T may be off by its own rounding, U[T] relative, plus what the
fp32 arithmetic in front of it loses. The losses are counted in roundings (EPS =
2^-24) of the terms that the formula adds up at that very entry, so that a small
gradient is held to a small error.
"""
from __future__ import annotations

import math

import pytest
import torch

from koemi_5hom_b200 import _native
from koemi_5hom_b200.cuda_kernels.dense import gated_recurrence
from koemi_5hom_b200.cuda_kernels.think import policy_loss
from oracle import training as plain

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


# ------------------------------------------------------- the gated recurrence

def recurrence_with_bounds(x, h0, gs, gf, valid=None, restart=None, low=plain.LOW, high=plain.HIGH):
    """64-bit (states, final, gradient of x, gradient of h0), and what fp32 may lose of each, position by position.

    a and k: ex2, rcp and four products, at most 16 roundings of s and of 1. A
    step adds a's and k's losses and three roundings of its terms to a times the
    loss so far; the walks over tiles round the same terms once more: all
    counted twice. The adjoint likewise, with |g| in place of g.
    """
    x, h0, gs, gf = x.double(), h0.double(), gs.double(), gf.double()
    features = x.shape[2] // 2
    p, c = x[..., :features], x[..., features:]
    span = high - low
    s, k = torch.sigmoid(p), torch.tanh(c)
    a = low + span * s
    live = torch.ones_like(a, dtype=torch.bool) if valid is None else valid[..., None].expand_as(a)
    cut = torch.zeros_like(live) if restart is None else restart[..., None].expand_as(a)
    keep = torch.where(live, a, 1.0)
    a_lost, k_lost = 16 * EPS * span * s + 2 * EPS * a, torch.full_like(k, 16 * EPS)
    h, lost = h0, torch.zeros_like(h0)
    states, states_lost, before, before_lost = [], [], [], []
    for t in range(x.shape[1]):
        h, lost = torch.where(cut[:, t], 0.0, h), torch.where(cut[:, t], 0.0, lost)
        before.append(h)
        before_lost.append(lost)
        size = h.abs() + k[:, t].abs()
        step = 2 * (a_lost[:, t] * size + (1 - a[:, t]) * k_lost[:, t] + 5 * EPS * size)
        lost = torch.where(live[:, t], a[:, t] * lost + step, lost)
        h = torch.where(live[:, t], a[:, t] * h + (1 - a[:, t]) * k[:, t], h)
        states.append(h)
        states_lost.append(lost)
    back, size, lost = gf, gf.abs(), torch.zeros_like(gf)
    dx, dx_lost = torch.zeros_like(x), torch.zeros_like(x)
    for t in range(x.shape[1] - 1, -1, -1):
        adjoint, size = gs[:, t] + back, gs[:, t].abs() + size
        lost = lost + 6 * EPS * size
        gap, gap_lost = before[t] - k[:, t], before_lost[t] + k_lost[:, t] + 2 * EPS * (before[t].abs() + k[:, t].abs())
        slope = span * s[:, t] * (1 - s[:, t])
        slope_lost = 20 * EPS * span * s[:, t]
        dp, dc = adjoint * gap * slope, adjoint * (1 - a[:, t]) * (1 - k[:, t] ** 2)
        dp_lost = lost * gap.abs() * slope + adjoint.abs() * (gap_lost * slope + gap.abs() * slope_lost)
        dc_lost = lost * (1 - a[:, t]) + adjoint.abs() * (a_lost[:, t] + 2 * EPS + (1 - a[:, t]) * 2 * (k_lost[:, t] + 2 * EPS))
        for part, exact, off in ((slice(0, features), dp, dp_lost), (slice(features, None), dc, dc_lost)):
            dx[:, t, part] = torch.where(live[:, t], exact, 0.0)
            dx_lost[:, t, part] = torch.where(live[:, t], off + 8 * EPS * exact.abs(), 0.0)
        lost = torch.where(cut[:, t], 0.0, keep[:, t] * lost + torch.where(live[:, t], 2 * a_lost[:, t] * size, 0.0))
        back, size = torch.where(cut[:, t], 0.0, keep[:, t] * adjoint), torch.where(cut[:, t], 0.0, keep[:, t] * size)
    stack = lambda rows: torch.stack(rows, 1)  # noqa: E731
    return ((stack(states), stack(states_lost)), (h, states_lost[-1]), (dx, dx_lost), (back, lost + 6 * EPS * size))


def check_recurrence(x, h0, gs, gf, valid=None, restart=None, low=plain.LOW, high=plain.HIGH):
    xg, hg = x.clone().requires_grad_(True), h0.clone().requires_grad_(True)
    states, final = gated_recurrence(xg, hg, valid=valid, restart=restart, minimum_retention=low, maximum_retention=high)
    got = (states, final, *torch.autograd.grad((states, final), (xg, hg), (gs, gf)))
    for result, (exact, lost) in zip(got, recurrence_with_bounds(x, h0, gs, gf, valid, restart, low, high)):
        check(result, exact, lost)


def recurrence_case(batch, length, features, dtype, seed, masks, cuda):
    g = torch.Generator().manual_seed(seed)
    x = (1.5 * torch.randn(batch, length, 2 * features, generator=g)).to(dtype).to(cuda)
    h0 = torch.randn(batch, features, generator=g).tanh().to(cuda)
    gs, gf = torch.randn(batch, length, features, generator=g).to(dtype).to(cuda), torch.randn(batch, features, generator=g).to(cuda)
    valid = (torch.rand(batch, length, generator=g) < 0.8).to(cuda) if masks else None
    restart = (torch.rand(batch, length, generator=g) < 0.05).to(cuda) if masks else None
    return x, h0, gs, gf, valid, restart


# exact in fp32, so that the kernel's bounds are the formula's
RETENTIONS = [(0.5, 0.5), (0.5, 0.5 + 2.0 ** -10), (0.875, 0.9375)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("length", [1, 16, 17, 300])
@pytest.mark.parametrize("low,high", RETENTIONS)
def test_recurrence_of_equal_and_narrow_retention_bounds(low, high, length, dtype, cuda):
    """Equal bounds: a is the bound and dp is 0. Narrow ones: the slope (hi - lo) s (1 - s) keeps its digits."""
    check_recurrence(*recurrence_case(3, length, 72, dtype, length, False, cuda), low=low, high=high)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("length", [3, 40])
def test_recurrence_of_small_candidates(length, dtype, cuda):
    """A candidate near 0 is as good as one near 1, and one of exactly 0 adds exactly nothing. Bounds of one half make
    every state half its candidate, each at a restart. 16-bit candidates below 2^-8 are their own tanh to 2^-17; from
    there on the 16 roundings of k (as above) are 2^-12 of it; fp32 takes the series, a few roundings of k itself."""
    g = torch.Generator().manual_seed(length)
    p = 3 * torch.randn(2, length, 64, generator=g)
    c = torch.randn(2, length, 64, generator=g) * torch.exp2(torch.randint(-23, -2, (2, length, 64), generator=g).float())
    c[:, :, ::5] = 0.0
    x = torch.cat((p, c), -1).to(dtype).to(cuda)
    every = torch.ones(2, length, dtype=torch.bool, device=cuda)
    states, _ = gated_recurrence(x, restart=every, minimum_retention=0.5, maximum_retention=0.5)
    exact = 0.5 * torch.tanh(x[..., 64:].double())
    check(states, exact, (2.0 ** -12 if dtype != torch.float32 else 16 * EPS) * exact.abs())
    assert not states[:, :, ::5].any()


@pytest.mark.parametrize("length", [1, 16, 64, 600])
@pytest.mark.parametrize("dtype", DTYPES)
def test_recurrence_of_zeros_stays_zero(dtype, length, cuda):
    """Zero projections leave a zero state at zero, whatever the gates."""
    x = torch.zeros(2, length, 2 * 64, device=cuda)
    x[..., :64] = torch.linspace(-6, 6, 64, device=cuda)
    states, final = gated_recurrence(x.to(dtype))
    assert not states.any() and not final.any()


@pytest.mark.parametrize("masks", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(3, 1, 64), (2, 8, 33), (3, 16, 40), (2, 17, 64), (1, 129, 515), (3, 200, 64), (2, 511, 72),
                                   (1, 1025, 96), (1, 2100, 64), (40, 130, 136)])
def test_recurrence_entry_by_entry(shape, dtype, masks, cuda):
    check_recurrence(*recurrence_case(*shape, dtype, 100 + sum(shape), masks, cuda))


def test_recurrence_of_clusters_entry_by_entry(cuda):
    """A few long chains, which clusters of CTAs walk, exchanging their tiles' maps in every wave."""
    for masks in (False, True):
        check_recurrence(*recurrence_case(1, 9000, 64, torch.bfloat16, 31, masks, cuda))


# ------------------------------------------------------------- the policy loss

CLIP_LOW, CLIP_HIGH, BETA = 0.2, 0.3, 0.05


def policy_case(rows, vocab, dtype, seed, cuda, offset=0.0):
    """Ratios away from the clipping's edges, where the gradient jumps; `offset` moves all logits."""
    g = torch.Generator().manual_seed(seed)
    logits = (2.5 * torch.randn(rows, vocab, generator=g) + offset).to(dtype)
    targets = torch.randint(0, vocab, (rows,), generator=g)
    return finish_case(dict(logits=logits, targets=targets, valid=torch.arange(rows) % 5 != 1), g, cuda)


def finish_case(case, g, cuda):
    rows = case["targets"].numel()
    lp = torch.log_softmax(case["logits"].double(), -1).gather(-1, case["targets"][:, None])[:, 0]
    drift = 0.2 * torch.randn(rows, generator=g).double()
    for edge in (math.log(1 - CLIP_LOW), math.log(1 + CLIP_HIGH)):
        drift = torch.where((drift - edge).abs() < 1e-2, edge + 2e-2, drift)
    case.update(old=(lp - drift).float(), advantages=torch.randn(rows, generator=g),
                reference=(lp + 0.1 * torch.randn(rows, generator=g)).float())
    return {name: t.to(cuda) for name, t in case.items()}


def policy_of(case, logits):
    return policy_loss(logits, case["targets"], case["old"], case["advantages"], reference_log_probs=case["reference"],
                       valid_mask=case["valid"], clip_low=CLIP_LOW, clip_high=CLIP_HIGH, kl_weight=BETA)


def policy_gradient_with_bounds(case, factor=1.0):
    """The 64-bit gradient, and what fp32 may lose of each of its entries.

    A log-prob loses the roundings of its exponentials' arguments and of their
    sum, 136 EPS in all; the ratio and e^d inherit that; an entry's probability
    loses the same, relative to itself.
    """
    x = case["logits"].double()
    live = case["valid"].double()
    count = max(1, int(case["valid"].sum()))
    p = torch.softmax(x, -1)
    lp = torch.log_softmax(x, -1).gather(-1, case["targets"][:, None])[:, 0]
    ratio, gap = torch.exp(lp - case["old"].double()), torch.exp(case["reference"].double() - lp)
    a = case["advantages"].double()
    free, clipped = ratio * a, ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * a
    slope = (torch.where(free <= clipped, -free, 0.0) + BETA * (1 - gap)) * live * factor / count
    slope_lost = 144 * EPS * ((ratio * a).abs() + BETA * (1 + gap)) * live * factor / count
    want = -slope[:, None] * p
    lost = p * (slope_lost + 144 * EPS * slope.abs())[:, None]
    at = case["targets"][:, None]
    return want.scatter_add(1, at, slope[:, None]), lost.scatter_add(1, at, slope_lost[:, None])


POLICY_SHAPES = [(64, 257), (17, 1024), (10, 4097), (7, 8200), (5, 32767), (6, 32768), (3, 65000), (2, 131072), (2, 250001), (2, 600001)]


def factor_of(dtype):
    return 64.0 if dtype == torch.float16 else 1.0  # fp16 gradients are there to be scaled


def gradient_of(case, logits=None, factor=1.0, **more):
    logits = case["logits"].clone().requires_grad_(True) if logits is None else logits
    result = policy_of(case, logits)
    return torch.autograd.grad(result.loss, logits, torch.tensor(factor, device=logits.device), **more)[0]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [900, 4097, 32768, 131072, 300000])
def test_policy_gradient_of_low_and_large_logits_in_every_backward(vocab, dtype, cuda):
    """Rows of the type's lowest value are uniform, and logits of large magnitude differ as they stand: in the first
    backward, and in another through a retained graph."""
    g = torch.Generator().manual_seed(vocab)
    most = torch.finfo(dtype).max
    logits = 2.5 * torch.randn(6, vocab, generator=g)
    logits[0] = -most
    logits[1] = torch.where(torch.arange(vocab) % 2 == 0, -most, most / 2)
    logits[3] += 3e4 if dtype == torch.float16 else 1e6
    logits[4] -= 200.0
    targets = torch.randint(0, vocab, (6,), generator=g) | 1  # odd: the entries of row 1 that are possible
    case = finish_case(dict(logits=logits.to(dtype), targets=targets.clamp_max(vocab - 1 - vocab % 2), valid=torch.ones(6, dtype=torch.bool)), g, cuda)
    factor = factor_of(dtype)
    leaf = case["logits"].clone().requires_grad_(True)
    result = policy_of(case, leaf)
    weight = torch.tensor(factor, device=cuda)
    want, lost = policy_gradient_with_bounds(case, factor)
    for retain in (True, True, False):
        got, = torch.autograd.grad(result.loss, leaf, weight, retain_graph=retain)
        check(got, want, lost)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [257, 4097, 32768, 131072])
def test_policy_gradient_is_rounded_once_whatever_the_factor(vocab, dtype, cuda):
    """A loss divided by the number of accumulated steps: 16-bit gradients are those of the formula, rounded once.
    An fp32 gradient is a product more, a rounding of 2^-24."""
    case = policy_case(9, vocab, dtype, vocab + 1, cuda)
    for factor in (1.0 / 3.0, 0.7):
        factor = torch.tensor(factor).item() * factor_of(dtype)  # as fp32 holds it
        want, lost = policy_gradient_with_bounds(case, factor)
        check(gradient_of(case, factor=factor), want, lost + (EPS * want.abs() if dtype == torch.float32 else 0.0))


def test_policy_entries_with_log_sum_exps_alone(cuda):
    """The C entries as a caller has them that keeps one float per row: the softmax is off by the log-sum-exps' rounding."""
    rows, vocab = 9, 1500
    case = policy_case(rows, vocab, torch.float32, 41, cuda)
    lib, stream = _native.library(), torch.cuda.current_stream().cuda_stream
    policy_of(case, case["logits"])  # initialises the device
    loss, kl, one = (torch.ones((), device=cuda) for _ in range(3))
    log_probs, lse, slopes = (torch.full((rows,), math.nan, device=cuda) for _ in range(3))
    size = lib.koemi_think_policy_loss_workspace()
    workspace, grad = torch.empty(size, dtype=torch.uint8, device=cuda), torch.full((rows, vocab), math.nan, device=cuda)
    at = lambda t: t.data_ptr()  # noqa: E731
    assert lib.koemi_think_policy_loss_forward(
        at(case["logits"]), rows, vocab, rows, 0, vocab, at(case["targets"]), at(case["old"]), at(case["advantages"]),
        at(case["reference"]), at(case["valid"]), CLIP_LOW, CLIP_HIGH, BETA, at(loss), at(kl), at(log_probs), at(lse), at(slopes),
        None, _native.F32, at(workspace), size, stream) == 0
    assert lib.koemi_think_policy_loss_backward(
        at(case["logits"]), rows, vocab, rows, 0, vocab, at(case["targets"]), at(case["valid"]), at(lse), at(slopes), at(one),
        at(grad), _native.F32, stream) == 0
    exact = torch.where(case["valid"], torch.logsumexp(case["logits"].double(), -1), 0.0)
    check(lse, exact, 136 * EPS)
    want, lost = policy_gradient_with_bounds(case)
    # a log-sum-exp below 32 rounds to 16 EPS once more
    check(grad, want, lost + 32 * EPS * want.abs())


def test_rescale_refuses_what_the_kernel_cannot_take(cuda):
    logits, targets = torch.zeros(6, 9, device=cuda, dtype=torch.bfloat16), torch.zeros(6, dtype=torch.int64, device=cuda)
    rows, one = torch.zeros(6, device=cuda), torch.ones((), device=cuda)
    policy_loss(logits, targets, rows, rows)  # registers the ops
    rescale, kept = torch.ops.koemi_b200.policy_loss_rescale, torch.ones(3, 6, device=cuda)
    for call in (lambda: rescale(logits[:5].clone(), logits, targets, None, kept, one),
                 lambda: rescale(logits.float(), logits, targets, None, kept, one),
                 lambda: rescale(logits.clone(), logits, targets[:5], None, kept, one),
                 lambda: rescale(logits.clone(), logits, targets, None, kept[:2], one),
                 lambda: rescale(logits.clone(), logits, targets, None, kept, rows)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", POLICY_SHAPES)
def test_policy_gradient_entry_by_entry(shape, dtype, cuda):
    case = policy_case(*shape, dtype, 7 + sum(shape), cuda)
    factor = factor_of(dtype)
    want, lost = policy_gradient_with_bounds(case, factor)
    got = gradient_of(case, factor=factor)
    check(got, want, lost)
    assert not got[~case["valid"]].any()
