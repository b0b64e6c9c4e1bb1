"""The operators around a training step, together: one block as it is trained
(pre-op, projection, per-head norms with rotation, attention, post-op, backward,
update of phi), the same step captured, and the debug-bounds build."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from mhc_ops_b200 import (NEWTON_SCHULZ_COEFFS, mhc_backward_manual, mhc_forward_pre, mhc_forward_pre_fused_norm,
                          mhc_muon_step, mhc_orthogonalize, mhc_post_fn, mhc_pre, mhc_qk_norm_rope,
                          mhc_qk_norm_rope_backward, mhc_qkv_norm_rope_fn)
from mhc_ops_b200.backward import param_grad_numel
from mhc_ops_b200.dist import DataParallelMHC
from mhc_ops_b200.synthetic import make_inputs
from oracle import train_oracle as O

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.gpu
B, S, n, D, HQ, HK, d = 2, 48, 4, 256, 4, 2, 64


def _block(seed=1):
    i = make_inputs(B, S, n, D, seed=seed).to("cuda")
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")   # noqa: E731
    return dict(x=i.x, phi=i.phi, alpha=i.alpha, bias=i.bias, wqkv=(rnd((HQ + 2 * HK) * d, D) / D ** 0.5).bfloat16(),
                wo=(rnd(D, HQ * d) / (HQ * d) ** 0.5).bfloat16(), wq=1 + 0.1 * rnd(d), wk=1 + 0.1 * rnd(d),
                inv_freq=(10000.0 ** (-torch.arange(d // 2, device="cuda") / (d // 2))).float(),
                target=rnd(B, S, n, D).bfloat16())


def _forward(t):
    h_in, h_post, h_res = mhc_pre(t["x"], t["phi"], t["alpha"], t["bias"])
    qkv = torch.nn.functional.linear(h_in, t["wqkv"]).view(B, S, HQ + 2 * HK, d)
    q, k, v = mhc_qkv_norm_rope_fn(qkv, HQ, HK, None, t["inv_freq"], t["wq"], t["wk"])
    k, v = (u.repeat_interleave(HQ // HK, dim=2) for u in (k, v))
    s = torch.einsum("bqhd,bkhd->bhqk", q.float(), k.float()) / d ** 0.5
    s = s.masked_fill(torch.ones(S, S, dtype=torch.bool, device="cuda").triu(1), float("-inf"))
    a = torch.einsum("bhqk,bkhd->bqhd", s.softmax(-1), v.float()).bfloat16().reshape(B, S, HQ * d)
    return mhc_post_fn(t["x"], h_res, h_post, torch.nn.functional.linear(a, t["wo"]))


def _forward64(t):
    """The block in float64 from the formulas (with the bf16 weights and streams as they are)."""
    x, phi = t["x"].double(), t["phi"]
    flat = x.reshape(B, S, n * D)
    mix = (flat @ phi.T) / torch.sqrt((flat * flat).mean(-1, keepdim=True) + 1e-6)
    pre, post, res = mix.split((n, n, n * n), dim=-1)
    al, bi = t["alpha"].double(), t["bias"].double()
    h_pre = torch.sigmoid(al[0] * pre + bi[:n]) + 1e-6
    h_post = 2 * torch.sigmoid(al[1] * post + bi[n:2 * n])
    h_res = (al[2] * res + bi[2 * n:]).view(B, S, n, n)
    h_in = (h_pre[..., None] * x).sum(2)
    qkv = (h_in @ t["wqkv"].double().T).view(B, S, HQ + 2 * HK, d)
    angle = O.angles(None, t["inv_freq"], B, S)
    q = O.norm_rope(qkv[:, :, :HQ], t["wq"].double(), None, angle, 1e-6, False)
    k = O.norm_rope(qkv[:, :, HQ:HQ + HK], t["wk"].double(), None, angle, 1e-6, False)
    k, v = (u.repeat_interleave(HQ // HK, dim=2) for u in (k, qkv[:, :, HQ + HK:]))
    s = torch.einsum("bqhd,bkhd->bhqk", q, k) / d ** 0.5
    s = s.masked_fill(torch.ones(S, S, dtype=torch.bool, device="cuda").triu(1), float("-inf"))
    a = torch.einsum("bhqk,bkhd->bqhd", s.softmax(-1), v).reshape(B, S, HQ * d)
    return (h_res @ x) + h_post[..., None] * (a @ t["wo"].double().T)[:, :, None]


def test_block_trains_a_step_like_float64():
    """phi's gradient through the whole block against float64, then its update.

    The block rounds to bf16 at ten places between x and the result (h_in, qkv,
    q, k, v, attention, y, out and their gradients), a relative 2^-8 each, on
    values that a projection or softmax averages over: 2^-8 sqrt(20) of the
    gradient's norm is a generous bound on their sum.
    """
    t = _block()
    t["phi"] = t["phi"].clone().requires_grad_()
    out = _forward(t)
    (out.float() * t["target"].float()).sum().backward()
    phi64 = t["phi"].detach().double().requires_grad_()
    (_forward64(dict(t, phi=phi64)) * t["target"].double()).sum().backward()
    err = (t["phi"].grad.double() - phi64.grad).norm() / phi64.grad.norm()
    assert err <= 20 ** 0.5 * 2.0 ** -8, float(err)
    # the update of the parameter with this gradient
    p0, g = t["phi"].detach().clone(), t["phi"].grad
    m = torch.zeros_like(p0)
    mhc_muon_step(t["phi"].detach(), g, m, 0.02, weight_decay=0.1)
    want, want_m = O.muon_step(p0, g, torch.zeros_like(p0), 0.02, 0.95, True, 0.1, 1.0, NEWTON_SCHULZ_COEFFS, 1e-7)
    # |O| <= 1.3 per singular direction; fp32 roundings of u lifted at most 485-fold (tests/test_muon_gpu.py)
    assert (t["phi"].detach() - want).norm() <= 0.02 * 3 * 2.0 ** -24 * 1100 * 24 ** 0.5 + 2.0 ** -22 * want.norm()
    assert (m - want_m).norm() <= 2.0 ** -22 * want_m.norm()


def test_row_factor_stands_in_for_the_norm_before_the_projection():
    """h_in_rstd of the fused norm, the norm's weight folded into the projection:
    the same q, k, v as normalising h_in first, up to the bf16 that this skips
    (one rounding of the normed row, 2^-8, through a projection's sum and the
    head's norm: at most 3 * 2^-8 of a head row's norm, and that of the output)."""
    t = _block(2)
    h_in, rstd, _, _ = mhc_forward_pre_fused_norm(t["x"], t["phi"], t["alpha"], t["bias"])
    w = 1 + 0.1 * torch.randn(D, device="cuda")
    folded = (t["wqkv"].float() * w).bfloat16()
    qkv = torch.nn.functional.linear(h_in, folded).view(B, S, -1, d)
    got = mhc_qk_norm_rope(qkv[:, :, :HQ], qkv[:, :, HQ:HQ + HK], None, t["inv_freq"], t["wq"], t["wk"],
                           v=qkv[:, :, HQ + HK:], row_scale=rstd)
    x = h_in.double()
    ref = ((x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6)) @ folded.double().T).view(B, S, -1, d)
    angle = O.angles(None, t["inv_freq"], B, S)
    want = [O.norm_rope(ref[:, :, :HQ], t["wq"].double(), None, angle, 1e-6, False),
            O.norm_rope(ref[:, :, HQ:HQ + HK], t["wk"].double(), None, angle, 1e-6, False), ref[:, :, HQ + HK:]]
    for a, b in zip(got, want):
        err = (a.double() - b).norm(dim=-1) / b.norm(dim=-1)
        assert err.max() <= 3 * 2.0 ** -8, float(err.max())


def test_row_factor_carries_its_gradient_to_h_in():
    """h_in's gradient through projection and row factor, dqkv w - drow_scale rstd^3 h_in / D, against float64 autograd.

    dqkv is right to (d/32 + 40) 2^-24 of its terms (tests/test_qkrope_gpu.py), the projection's sums of 512
    products add as much again as they have terms, at worst 512 2^-24 of the sum of magnitudes; the norms of the two
    sums differ from sqrt by less than 10: 1e-3 of the gradient's norm bounds all of it, and the row factor's part
    (eps is large here, so that it is not lost below that) is a tenth of the whole or more."""
    g = torch.Generator(device="cuda").manual_seed(7)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")   # noqa: E731
    eps, f = 0.3, (10000.0 ** (-torch.arange(d // 2, device="cuda") / (d // 2))).float()
    h, w = rnd(B, S, D), rnd((HQ + 2 * HK) * d, D) / D ** 0.5
    up = rnd(B, S, HQ + 2 * HK, d)
    rstd = 1.0 / torch.sqrt((h * h).mean(-1) + 1e-6)
    qkv = (h @ w.T).view(B, S, -1, d)
    parts = (HQ, HK, HK)
    q, k, v = qkv.split(parts, dim=2)
    dq, dk, dv = up.split(parts, dim=2)
    dqkv = torch.empty_like(qkv)
    out = mhc_qk_norm_rope_backward(q, k, None, f, dq, dk, v=v, dv_out=dv, row_scale=rstd, eps=eps,
                                    grad_out=dqkv.split(parts, dim=2))
    through = -out[5][..., None] * rstd[..., None] ** 3 * h / D
    got = dqkv.flatten(2) @ w + through
    x = h.double().requires_grad_()
    y = (x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6)) @ w.double().T
    y = y.view(B, S, -1, d)
    angle = O.angles(None, f, B, S)
    o = [O.norm_rope(y[:, :, :HQ], None, None, angle, eps, False),
         O.norm_rope(y[:, :, HQ:HQ + HK], None, None, angle, eps, False), y[:, :, HQ + HK:]]
    want, = torch.autograd.grad(torch.cat(o, dim=2), x, up.double())
    assert (got - want).norm() <= 1e-3 * want.norm()
    assert through.norm() >= 0.1 * want.norm() or (got - through - want).norm() >= 5e-3 * want.norm()


def test_calls_from_two_threads_on_two_streams():
    """Calls that overlap share nothing: each thread's results equal the same calls made alone."""
    import threading
    u = [torch.randn(4, 24, 3000, device="cuda"), torch.randn(3, 80, 700, device="cuda")]
    q = [torch.randn(2, 300, 4, 64, device="cuda").bfloat16() for _ in range(2)]
    f = torch.rand(32, device="cuda")

    def work(i):
        return (mhc_orthogonalize(u[i]),) + mhc_qk_norm_rope_backward(q[i], q[i], None, f, q[i], q[i], torch.ones(
            64, device="cuda"))[:4]

    alone = [work(0), work(1)]
    torch.cuda.synchronize()
    got = [None, None]

    def run(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                got[i] = work(i)
        s.synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(2):
        for a, b in zip(got[i], alone[i]):
            assert a is None and b is None or torch.equal(a, b)


def test_data_parallel_object_updates_phi():
    """Forward, backward and update through DataParallelMHC equal the calls by hand."""
    i = make_inputs(2, 64, 4, 256, seed=3).to("cuda")
    dp = DataParallelMHC(4, 256)
    phi, m = i.phi.clone(), torch.zeros_like(i.phi)
    fw = dp.forward(i.x, phi, i.alpha, i.bias)
    dp.backward(i.x, phi, i.alpha, i.bias, fw[3], fw[4], fw[5], fw[1], i.dh_in, i.dh_post, i.dh_res, i.gamma)
    dp.muon_step(phi, m, 0.02, weight_decay=0.1)
    phi2, m2 = i.phi.clone(), torch.zeros_like(i.phi)
    f2 = mhc_forward_pre(i.x, phi2, i.alpha, i.bias, outflag=True)
    g2 = mhc_backward_manual(i.x, phi2, i.alpha, i.bias, f2[3], f2[4], f2[5], f2[1], i.dh_in, i.dh_post, i.dh_res,
                             i.gamma)
    mhc_muon_step(phi2, g2[1], m2, 0.02, weight_decay=0.1)
    torch.cuda.synchronize()
    assert torch.equal(phi, phi2) and torch.equal(m, m2)
    assert dp.flat.numel() == param_grad_numel(4, 256)


def test_whole_step_captured_and_replayed():
    """Forward, backward and update in one graph: replays equal eager steps bit for bit."""
    def step(t, m):
        fw = mhc_forward_pre(t["x"], t["phi"], t["alpha"], t["bias"], outflag=True)
        qkv = torch.nn.functional.linear(fw[0], t["wqkv"]).view(B, S, HQ + 2 * HK, d)
        q, k = mhc_qk_norm_rope(qkv[:, :, :HQ], qkv[:, :, HQ:HQ + HK], None, t["inv_freq"], t["wq"], t["wk"])
        bw = mhc_backward_manual(t["x"], t["phi"], t["alpha"], t["bias"], fw[3], fw[4], fw[5], fw[1],
                                 q.reshape(B, S, -1)[..., :D], fw[1], fw[2], None)
        mhc_muon_step(t["phi"], bw[1], m, 0.02)
        return q, k

    t, m = _block(4), torch.zeros(n * n + 2 * n, n * D, device="cuda")
    e, em = {k: v.clone() for k, v in t.items()}, m.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step({k: v.clone() for k, v in t.items()}, m.clone())   # warm-up on the capturing stream
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        outs = step(t, m)
    for _ in range(3):
        graph.replay()
        ref = step(e, em)
    torch.cuda.synchronize()
    assert torch.equal(t["phi"], e["phi"]) and torch.equal(m, em)
    for a, b in zip(outs, ref):
        assert torch.equal(a, b)
    del graph


def test_captured_autograd_backward():
    """Forward and backward of the autograd wrapper in one graph.  torch ties a leaf's gradient node to the stream
    of the first live graph that uses the leaf, so no eager graph of the leaves may live through the capture: the
    warm-up's is dropped before it."""
    t = _block(5)
    qkv = torch.randn(B, S, HQ + 2 * HK, d, device="cuda").bfloat16().requires_grad_()
    w = t["wq"].clone().requires_grad_()
    up = torch.randn(B, S, HQ, d, device="cuda").bfloat16()
    run = lambda: mhc_qkv_norm_rope_fn(qkv, HQ, HK, None, t["inv_freq"], w, t["wk"])[0]   # noqa: E731
    want = torch.autograd.grad(run(), (qkv, w), up)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        grads = torch.autograd.grad(run(), (qkv, w), up)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(grads, want):
        assert torch.equal(a, b)
    del graph


def test_debug_bounds_build_sees_no_out_of_buffer_access_and_matches_normal_build(tmp_path):
    from mhc_ops_b200 import build

    dbg = build.build(debug_bounds=True)
    out = str(tmp_path / "dbg.npz")
    env = dict(os.environ, MHC_OPS_LIBRARY=dbg, PYTHONPATH=ROOT)
    res = subprocess.run([sys.executable, "-m", "tests._train_bounds_cases", out], cwd=ROOT, env=env,
                         capture_output=True, text=True, timeout=900)
    assert res.returncode == 0, f"debug-bounds run failed:\n{res.stdout[-3000:]}\n{res.stderr[-3000:]}"
    got = dict(np.load(out))
    from tests._train_bounds_cases import run_cases
    ref = run_cases(debug=False)
    assert set(ref) == set(got), sorted(set(ref) ^ set(got))
    for k in ref:
        same = ref[k].view(np.uint8) == got[k].view(np.uint8)
        assert same.all(), f"{k}: debug-bounds build differs in {int((~same).sum())} of {same.size} bytes"
