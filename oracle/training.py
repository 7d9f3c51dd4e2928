"""Plain 64-bit forms of the training operators (test infrastructure; see oracle/__init__.py).

Written from the formulas, position by position and row by row, on whatever
device the inputs are on.
"""
from __future__ import annotations

import torch

LOW, HIGH = 2.0 ** -8, 1.0 - 2.0 ** -8


def gated_recurrence(projections, initial=None, valid=None, restart=None, low=LOW, high=HIGH):
    """(states, final) of h_t = a h' + (1 - a) tanh(c), differentiable by autograd."""
    x = projections.double()
    batch, length, double = x.shape
    features = double // 2
    h = x.new_zeros(batch, features) if initial is None else initial.double()
    states = []
    for t in range(length):
        if restart is not None:
            h = torch.where(restart[:, t, None], torch.zeros_like(h), h)
        a = low + (high - low) * torch.sigmoid(x[:, t, :features])
        new = a * h + (1 - a) * torch.tanh(x[:, t, features:])
        h = new if valid is None else torch.where(valid[:, t, None], new, h)
        states.append(h)
    return (torch.stack(states, 1) if states else x.new_zeros(batch, 0, features)), h


def route_learned(logits, valid, top_k, renormalize):
    """(ids, weights, counts, balance), weights and balance differentiable by autograd."""
    x = logits.double()
    tokens, experts = x.shape
    live = ~(x == -torch.inf).all(-1)
    if valid is not None:
        live = live & valid
    safe = torch.where(live[:, None], x, torch.zeros_like(x))
    p = torch.softmax(safe, -1)
    ranked = torch.sort(torch.where(torch.isnan(safe), -torch.inf, safe), dim=-1, descending=True, stable=True).indices[:, :top_k]
    weights = p.gather(-1, ranked)
    if renormalize:
        weights = weights / weights.sum(-1, keepdim=True)
    counts = torch.bincount(ranked[live].reshape(-1), minlength=experts)
    n = max(1, int(live.sum()))
    importance = torch.where(live[:, None], p, torch.zeros_like(p)).sum(0) / n
    balance = experts * (importance * (counts.double() / max(1, int(counts.sum())))).sum()
    ids = torch.where(live[:, None], ranked, torch.full_like(ranked, -1))
    return ids, torch.where(live[:, None], weights, torch.zeros_like(weights)), counts, balance


def policy_loss(logits, targets, old, advantages, reference=None, valid=None, clip_low=0.2, clip_high=0.2, beta=0.0):
    """(loss, kl, log_probs), the loss differentiable by autograd."""
    live = torch.ones_like(targets, dtype=torch.bool) if valid is None else valid
    x = torch.where(live[..., None], logits.double(), torch.zeros_like(logits, dtype=torch.float64))
    target = torch.where(live, targets, torch.zeros_like(targets))
    lp = torch.log_softmax(x, -1).gather(-1, target[..., None])[..., 0]
    zero = torch.zeros_like(lp)
    keep = lambda t: torch.where(live, t.double(), zero)  # noqa: E731
    ratio = torch.exp(lp - keep(old))
    a = keep(advantages)
    free, clipped = ratio * a, ratio.clamp(1 - clip_low, 1 + clip_high) * a
    loss = -torch.where(free <= clipped, free, clipped)
    kl = zero
    if reference is not None:
        d = keep(reference) - lp
        kl = torch.expm1(d) - d
        loss = loss + beta * kl
    n = max(1, int(live.sum()))
    return torch.where(live, loss, zero).sum() / n, torch.where(live, kl, zero).sum() / n, torch.where(live, lp, zero)


def clip_gradients(gradients, max_norm):
    """(norm, clipped gradients)."""
    norm = torch.stack([g.double().square().sum() for g in gradients]).sum().sqrt()
    return norm, [g.double() * min(1.0, max_norm / (float(norm) + 1e-6)) for g in gradients]
