"""Plain 64-bit forms of the feed-forward sub-layer's operators (test infrastructure; see oracle/__init__.py).

Written from the formulas, differentiable by autograd, on whatever device the
inputs are on.
"""
from __future__ import annotations

import numpy as np
import torch

_GOLDEN = 0x9E3779B97F4A7C15


def layer_norm(values, weight, bias=None, eps=1e-5):
    x = values.double()
    centred = x - x.mean(-1, keepdim=True)
    y = centred / (centred.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    return y if bias is None else y + bias.double()


def _mix(z):
    """SplitMix64's finaliser on a uint64 array."""
    z = z + np.uint64(_GOLDEN)
    z = (z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
    z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
    return z ^ (z >> np.uint64(31))


def dropout_lanes(first, count, seed, site, step):
    """The 16 bits of values ``first`` .. ``first + count - 1``."""
    word = lambda v: np.array([v], dtype=np.uint64)  # noqa: E731
    with np.errstate(over="ignore"):
        key = _mix(word(seed) ^ _mix(word(site) ^ _mix(word(step))))
        e = np.arange(first, first + count, dtype=np.uint64)
        words = _mix(key + (e >> np.uint64(2)) * np.uint64(_GOLDEN))
    return ((words >> (np.uint64(16) * (e & np.uint64(3)))) & np.uint64(0xFFFF)).astype(np.int64)


def dropout(values, probability, seed, site=0, step=0, residual=None):
    dropped = int(probability * 65536 + 0.5)
    lanes = torch.from_numpy(dropout_lanes(0, values.numel(), seed, site, step)).to(values.device).view(values.shape)
    scaled = values.double() * (65536.0 / (65536 - dropped) if dropped < 65536 else 0.0)
    y = torch.where(lanes < dropped, torch.zeros_like(scaled), scaled)
    return y if residual is None else residual.double() + y


def gated_feed_forward(values, gate_weight, value_weight, output_weight, gate_bias=None, value_bias=None, output_bias=None):
    def project(x, weight, bias):
        y = x @ weight.double().T
        return y if bias is None else y + bias.double()

    x = values.double()
    gate = project(x, gate_weight, gate_bias)
    return project(gate * torch.sigmoid(gate) * project(x, value_weight, value_bias), output_weight, output_bias)
