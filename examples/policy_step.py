"""Policy tuning of a small recurrent mixture-of-experts model on the training operators.

One step: gate projections -> gated recurrence -> learned route with its balance
loss -> experts -> head logits -> clipped policy loss with a KL term against the
starting policy -> backward -> clipping by the global norm -> SGD. Answers are
sampled from the current policy one token at a time, with the recurrence's
single-token form; the reward is the share of even tokens.

    python examples/policy_step.py --steps 20
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch
from torch import Tensor, nn

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from koemi_5hom_b200.cuda_kernels.core import clip_gradients  # noqa: E402
from koemi_5hom_b200.cuda_kernels.dense import gated_recurrence  # noqa: E402
from koemi_5hom_b200.cuda_kernels.moe import route_learned_topk  # noqa: E402
from koemi_5hom_b200.cuda_kernels.think import policy_loss  # noqa: E402

VOCABULARY, WIDTH, EXPERTS, TOP_K = 257, 128, 8, 2
CLIP_LOW, CLIP_HIGH, KL_WEIGHT, BALANCE_WEIGHT, MAX_NORM = 0.2, 0.28, 0.02, 0.01, 1.0


class Policy(nn.Module):
    """Embedding, one gated recurrence, one routed layer of gated experts, a head."""

    def __init__(self) -> None:
        super().__init__()
        self.embedding = nn.Embedding(VOCABULARY, WIDTH)
        self.gates = nn.Linear(WIDTH, 2 * WIDTH)
        self.router = nn.Linear(WIDTH, EXPERTS, bias=False)
        self.experts_in = nn.Parameter(torch.randn(EXPERTS, WIDTH, 2 * WIDTH) / WIDTH ** 0.5)
        self.experts_out = nn.Parameter(torch.randn(EXPERTS, WIDTH, WIDTH) / WIDTH ** 0.5)
        self.head = nn.Linear(WIDTH, VOCABULARY)

    def forward(self, ids: Tensor, state: Tensor | None = None, valid: Tensor | None = None) -> tuple[Tensor, Tensor, Tensor]:
        """(logits [batch, length, vocabulary], final state, balance loss)."""
        hidden, state = gated_recurrence(self.gates(self.embedding(ids)), state, valid=valid)
        rows = hidden.reshape(-1, WIDTH)
        route = route_learned_topk(self.router(rows), None if valid is None else valid.reshape(-1), top_k=TOP_K, renormalize=True)
        # a few small experts: every one on every row, weighted by the route
        weight = torch.zeros(rows.shape[0], EXPERTS, device=rows.device).scatter_add(1, route.expert_ids.clamp_min(0), route.weights)
        gate, value = torch.einsum("nd,edf->nef", rows, self.experts_in).chunk(2, -1)
        mixed = torch.einsum("nef,efd,ne->nd", nn.functional.silu(gate) * value, self.experts_out, weight)
        return self.head(rows + mixed).reshape(*ids.shape, VOCABULARY), state, route.balance_loss


def log_probs_of(logits: Tensor, targets: Tensor) -> Tensor:
    """The targets' log-probs: the policy loss without advantages."""
    zeros = torch.zeros(targets.shape, device=logits.device)
    return policy_loss(logits, targets, zeros, zeros).log_probs


@torch.no_grad()
def sample(model: Policy, batch: int, length: int, generator: torch.Generator) -> Tensor:
    """Answers [batch, length + 1] that start with token 0, a token at a time."""
    device = model.head.weight.device
    ids, state, answer = torch.zeros(batch, 1, dtype=torch.int64, device=device), None, []
    for _ in range(length):
        answer.append(ids)
        logits, state, _ = model(ids, state)
        ids = torch.multinomial(torch.softmax(logits[:, 0], -1), 1, generator=generator)
    return torch.cat((*answer, ids), 1)


def train(steps: int, batch: int = 64, length: int = 48, seed: int = 0, rate: float = 2.0, report=None) -> list[float]:
    """Mean rewards per step."""
    torch.manual_seed(seed)
    device = torch.device("cuda", torch.cuda.current_device())
    generator = torch.Generator(device).manual_seed(seed)
    model, start = Policy().to(device), Policy().to(device)
    start.load_state_dict(model.state_dict())
    rewards = []
    for step in range(steps):
        answers = sample(model, batch, length, generator)
        inputs, targets = answers[:, :-1], answers[:, 1:]
        lengths = torch.randint(length // 2, length + 1, (batch, 1), generator=generator, device=device)
        valid = torch.arange(length, device=device) < lengths
        reward = (targets % 2 == 0).float()
        advantages = reward - (reward * valid).sum() / valid.sum()
        with torch.no_grad():
            old = log_probs_of(model(inputs, valid=valid)[0], targets)
            reference = log_probs_of(start(inputs, valid=valid)[0], targets)
        for _ in range(2):  # the second pass has ratios away from one
            model.zero_grad(set_to_none=True)
            logits, _, balance = model(inputs, valid=valid)
            result = policy_loss(logits, targets, old, advantages, reference_log_probs=reference, valid_mask=valid,
                                 clip_low=CLIP_LOW, clip_high=CLIP_HIGH, kl_weight=KL_WEIGHT)
            (result.loss + BALANCE_WEIGHT * balance).backward()
            gradients = [p.grad for p in model.parameters()]
            norm = clip_gradients(gradients, MAX_NORM)
            with torch.no_grad():
                for p in model.parameters():
                    p.sub_(p.grad, alpha=rate)
        rewards.append(float((reward * valid).sum() / valid.sum()))
        if report:
            report(f"step {step}: reward {rewards[-1]:.3f}  loss {result.loss.item():+.4f}  kl {result.kl.item():.4f}  "
                   f"balance {balance.item():.3f}  norm {norm.item():.3f}")
    return rewards


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=20)
    train(parser.parse_args().steps, report=print)
