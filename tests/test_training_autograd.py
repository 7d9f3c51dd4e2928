"""The training operators in torch's own machinery, on meta tensors: nothing is computed, everything is recorded."""
from __future__ import annotations

import subprocess
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent


def test_first_calls_from_several_threads():
    """Both threads come to the registration before either has finished it."""
    code = """
import threading, time
from koemi_5hom_b200 import _native
from koemi_5hom_b200.cuda_kernels import _training
binding, errors = _native.binding, []
def slow():
    time.sleep(0.5)
    return binding()
_native.binding = slow
import torch
_native.ensure_device = lambda device: None
def call():
    try:
        _training.load(torch.device("cuda", 0))
    except Exception as error:
        errors.append(error)
threads = [threading.Thread(target=call) for _ in range(4)]
for t in threads: t.start()
for t in threads: t.join()
assert not errors, errors
assert _training.loaded()
"""
    result = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert result.returncode == 0, result.stderr
