"""The examples run as a user runs them."""
from __future__ import annotations

import importlib.util
import math
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parent.parent


def test_policy_step_learns():
    """Rewards start at the share of even tokens (a half) and rise: 1024 valid
    answers' tokens a step leave a standard error below 0.02."""
    spec = importlib.util.spec_from_file_location("policy_step", ROOT / "examples" / "policy_step.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    rewards = example.train(12)
    assert all(math.isfinite(r) for r in rewards)
    assert abs(rewards[0] - 0.5) < 0.1 and rewards[-1] > rewards[0] + 0.1
