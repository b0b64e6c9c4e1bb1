"""Calls of the operators around a training step that the documentation allows and a single thread, a warm process
or a plain layout never makes."""
import os
import subprocess
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.gpu


def test_first_backwards_of_a_process_take_any_size():
    """rot + 2 d = 1536: with their static arrays these take a little more shared memory than a kernel has without
    asking.  In a process of its own, since an earlier, wider call would have raised the kernel's limit.  The last
    rows start off a 16-byte boundary."""
    code = """
import torch
from tests.test_qkrope_gpu import _check, _inputs
for d, rot, off in ((768, 0, 0), (640, 256, 0), (704, 128, 0), (512, 512, 1)):
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        t = _inputs(2, 5, 3, 2, 1, d, rot, dtype, seed=3)
        flat = torch.empty(t["qkv"].numel() + off, dtype=dtype, device="cuda")[off:].view(t["qkv"].shape)
        flat.copy_(t["qkv"])
        t["q"], t["k"], t["v"] = flat.split((3, 2, 1), dim=2)
        for interleaved in (False, True):
            _check(t, rot, interleaved=interleaved)
"""
    res = subprocess.run([sys.executable, "-c", code], cwd=ROOT, env=dict(os.environ, PYTHONPATH=ROOT),
                         capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stderr[-2000:]
