"""The operators around a training step under torch.compile: whole graphs, the eager calls' bits, no warning.

Traced without code generation (backend aot_eager), which runs the same operators."""
import os
import subprocess
import sys
import warnings

import pytest
import torch

from mhc_ops_b200 import (mhc_muon_step, mhc_orthogonalize, mhc_qk_norm_rope, mhc_qk_norm_rope_backward,
                          mhc_qk_norm_rope_fn, mhc_qkv_norm_rope_fn, ops)

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.gpu
B, S, HQ, HK, d = 2, 30, 4, 2, 64


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


F = lambda: torch.rand(d // 2, device="cuda", generator=torch.Generator(device="cuda").manual_seed(9))   # noqa: E731


@pytest.mark.parametrize("twice", [False, True])
def test_packed_projection_and_its_gradients(twice):
    """With one weight for queries and keys its gradient is the sum of both."""
    def fn(qkv, f, wq, wk, sc):
        q, k, v = mhc_qkv_norm_rope_fn(qkv, HQ, HK, None, f, wq, wk, row_scale=sc)
        return (q.float() ** 2).sum() + k.float().sum() * 3 + (v.float() ** 3).sum()

    qkv, sc, wq = _leaf(B, S, HQ + 2 * HK, d, dtype=torch.bfloat16), _leaf(B, S, seed=1), _leaf(d, seed=2)
    wk = wq if twice else _leaf(d, seed=3)
    leaves = (qkv, sc, wq) if twice else (qkv, sc, wq, wk)
    want = torch.autograd.grad(fn(qkv, F(), wq, wk, sc), leaves)
    _same(torch.autograd.grad(_compiled(fn)(qkv, F(), wq, wk, sc), leaves), want)


def test_one_tensor_for_queries_keys_and_values():
    def fn(q, k, v, f, w, u):
        q, k, v = mhc_qk_norm_rope_fn(q, k, None, f, w, u, v=v)
        return (q.float() ** 3).sum() + k.float().sum() * 3 + (v.float() ** 2).sum()

    x, w = _leaf(B, S, HQ, d), _leaf(d, seed=2)
    want = torch.autograd.grad(fn(x, x, x, F(), w, w), (x, w))
    apart = [t.detach().clone().requires_grad_() for t in (x, x, x, w, w)]
    parts = torch.autograd.grad(fn(*apart[:3], F(), *apart[3:]), apart)
    for got, p in ((want[0], parts[:3]), (want[1], parts[3:])):   # the same terms, added in 32 bits
        assert (got - sum(t.double() for t in p)).abs().max() <= 2 ** -22 * sum(t.abs().max() for t in p)
    _same(torch.autograd.grad(_compiled(fn)(x, x, x, F(), w, w), (x, w)), want)


def test_calls_by_hand():
    def by_hand(q, k, f, up_q, up_k, w):
        y, z = mhc_qk_norm_rope(q, k, None, f, w)
        pack = torch.empty(B, S, HQ + HK, d, device="cuda", dtype=q.dtype)
        out = mhc_qk_norm_rope_backward(q, k, None, f, up_q, up_k, w, grad_out=pack.split((HQ, HK), dim=2))
        apart = mhc_qk_norm_rope_backward(q, k, None, f, up_q, up_k, w)
        return y, z, pack * 1, out[0] * 1, out[3], apart[0], apart[3]

    rnd = lambda h, s: _leaf(B, S, h, d, dtype=torch.bfloat16, seed=s).detach()   # noqa: E731
    args = (rnd(HQ, 1), rnd(HK, 2), F(), rnd(HQ, 3), rnd(HK, 4), _leaf(d, seed=5).detach())
    _same(_compiled(by_hand)(*args), by_hand(*args))

    def short(q, k, f):
        return mhc_qk_norm_rope_backward(q, k, None, f, q, k, grad_out=(torch.empty_like(q),))

    with pytest.raises(Exception, match="hold 2"):
        _compiled(short)(args[0], args[1], args[2])


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
