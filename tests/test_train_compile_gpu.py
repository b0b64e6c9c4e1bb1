"""The operators around a training step under torch.compile: whole graphs, the eager calls' bits, no warning.

Traced without code generation (backend aot_eager), which runs the same operators."""
import os
import subprocess
import sys
import warnings

import pytest
import torch

from mhc_ops_b200 import mhc_muon_step, mhc_orthogonalize, ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.gpu


def _compiled(fn):
    ops.load()
    return torch.compile(fn, backend="aot_eager", fullgraph=True)


def _same(got, want):
    assert len(got) == len(want)
    for i, (a, b) in enumerate(zip(got, want)):
        assert torch.equal(a, b), i


def _leaf(*shape, dtype=torch.float32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype).requires_grad_()


def test_update_and_orthogonalisation_of_lists():
    new = lambda s: [_leaf(8, 64, seed=s + i).detach() for i in range(3)]   # noqa: E731

    def step(ps, gs, ms):
        mhc_muon_step(ps, gs, ms, 0.1)
        return [p * 1 for p in ps]

    with warnings.catch_warnings():
        warnings.filterwarnings("error", message=".*alias.*")
        p, g, m = new(0), new(10), new(20)
        p2, m2 = [t.clone() for t in p], [t.clone() for t in m]
        out = _compiled(step)(p, g, m)
        step(p2, g, m2)
        _same(list(out) + p + m, p2 + p2 + m2)
        _same(_compiled(lambda gs: mhc_orthogonalize(gs))(g), mhc_orthogonalize(g))
        _same([_compiled(lambda t: mhc_orthogonalize(t))(g[0])], [mhc_orthogonalize(g[0])])


def test_first_use_of_a_process_may_be_inside_a_compiled_function():
    """Behind ops.load(): an operator's first call is traced like any other."""
    code = """
import torch
from mhc_ops_b200 import mhc_muon_step, mhc_orthogonalize, mhc_qk_norm_rope_fn, ops
ops.load()
def fn(q, k, f, g, p, m):
    y = mhc_qk_norm_rope_fn(q, k, None, f)[0]
    mhc_muon_step(p, g, m, 0.1)
    return y, mhc_orthogonalize(g)
q, k = torch.randn(1, 3, 2, 16, device="cuda", requires_grad=True), torch.randn(1, 3, 1, 16, device="cuda")
f, g = torch.rand(8, device="cuda"), torch.randn(8, 64, device="cuda")
p, m = torch.randn(8, 64, device="cuda"), torch.zeros(8, 64, device="cuda")
y, o = torch.compile(fn, backend="aot_eager", fullgraph=True)(q, k, f, g, p.clone(), m.clone())
dq, = torch.autograd.grad(y.sum(), q)
z, r = fn(q, k, f, g, p, m)
assert torch.equal(y, z) and torch.equal(o, r) and torch.equal(dq, torch.autograd.grad(z.sum(), q)[0])
"""
    res = subprocess.run([sys.executable, "-c", code], cwd=ROOT, env=dict(os.environ, PYTHONPATH=ROOT),
                         capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stderr[-2000:]
