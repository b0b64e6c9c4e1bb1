"""Calls of the operators around a training step that the documentation allows and a single thread, a warm process
or a plain layout never makes."""
import ctypes
import os
import subprocess
import sys
import threading

import pytest
import torch

from mhc_ops_b200 import _lib, mhc_muon_step, mhc_orthogonalize, mhc_qk_norm_rope_backward

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


def _matrix_call(C):
    """mhc_orthogonalize of one 8 x C matrix (one launch, shared memory by C) on a stream of its own."""
    u = torch.randn(8, C, device="cuda", generator=torch.Generator(device="cuda").manual_seed(C))
    out, s = torch.empty_like(u), torch.cuda.Stream()
    co = (ctypes.c_double * 3)(1.5, -0.5, 0.0)
    src, dst = (ctypes.c_void_p * 1)(u.data_ptr()), (ctypes.c_void_p * 1)(out.data_ptr())
    vp = lambda x: ctypes.cast(x, ctypes.c_void_p)   # noqa: E731
    a = _lib.OrthoArgs(inp=vp(src), out=vp(dst), count=1, rows=8, cols=C, dtype=2, steps=1, coeffs=vp(co), eps=1e-7)
    return (lambda: _lib.load().mhc_orthogonalize(ctypes.byref(a), s.cuda_stream)), out, s, (u, co, src, dst)


def _row_call(d):
    """mhc_qk_norm_rope_bwd of one token of d elements off the vector kernels (shared memory by d)."""
    x = torch.randn(1, 1, 2, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(d))
    out, dk, dw, s = torch.empty_like(x), torch.empty_like(x), torch.empty(d, device="cuda"), torch.cuda.Stream()
    ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    heads = lambda t: _lib.Heads(t.data_ptr(), *t.stride()[:3])   # noqa: E731
    a = _lib.QkArgs(q=heads(x), k=heads(x), batch=1, seq=1, q_heads=2, k_heads=2, d=d, rot=0, dtype=2, eps=1e-6)
    b = _lib.QkBwdArgs(fwd=a, dq_out=heads(x), dk_out=heads(x), dq=heads(out), dk=heads(dk), dq_weight=dw.data_ptr(),
                       workspace=ws.data_ptr(), workspace_bytes=ws.numel())
    return (lambda: _lib.load().mhc_qk_norm_rope_bwd(ctypes.byref(b), s.cuda_stream)), out, s, (x, dk, dw, ws)


@pytest.mark.parametrize("make,sizes", [(_matrix_call, (4000, 2000)), (_row_call, (1024, 800))])
def test_two_threads_with_two_sizes_of_one_kernel(make, sizes):
    """Each thread's calls all succeed: what a kernel may take of shared memory is the process's, not the call's."""
    calls = [make(n) for n in sizes]
    alone = []
    for call, out, s, _ in calls:
        s.wait_stream(torch.cuda.current_stream())
        assert call() == 0
        s.synchronize()
        alone.append(out.clone())
    torch.cuda.synchronize()
    refused = [0, 0]

    def run(i):
        torch.cuda.set_device(0)
        for _ in range(5000):
            refused[i] += calls[i][0]() != 0

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert refused == [0, 0]
    for (_, out, _, _), want in zip(calls, alone):
        assert torch.equal(out, want)


@pytest.mark.parametrize("L,R,C", [(1, 8, 1024), (1, 24, 512), (2, 24, 4096), (40, 35, 700), (3, 40, 2048)])
def test_repeated_calls_beside_other_work_return_the_same_bytes(L, R, C):
    """The iteration by blocks of the lower triangle, whose results and mirror images have one writer each."""
    u = torch.randn(L, R, C, device="cuda", generator=torch.Generator(device="cuda").manual_seed(R))
    other, x = torch.cuda.Stream(), torch.randn(2048, 2048, device="cuda")
    want = mhc_orthogonalize(u)
    torch.cuda.synchronize()
    outs = []
    for i in range(40):
        with torch.cuda.stream(other):
            for _ in range(i % 4):
                x.mul_(1.0)
        outs.append(mhc_orthogonalize(u))
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, want)


@pytest.mark.parametrize("L,R,C", [(64, 24, 4099), (3, 24, 16384), (6, 35, 10005), (2, 63, 4097), (5, 80, 2051),
                                   (1, 80, 32768), (2, 8, 1000)])
def test_update_applies_the_momentum_it_wrote(L, R, C):
    """Without nesterov, decay and parameter the update is -orthogonalised(new momentum), by the same kernels in the
    same order: the same bits, unless the application read a momentum from before the call.  Odd widths let rows of
    two CTAs share a cache line."""
    g = torch.Generator(device="cuda").manual_seed(C)
    m = torch.randn(L, R, C, device="cuda", generator=g)
    for _ in range(10):
        grad = torch.randn(L, R, C, device="cuda", generator=g)
        p = torch.zeros(L, R, C, device="cuda")
        mhc_muon_step(p, grad, m, 1.0, momentum=0.5, nesterov=False)
        assert torch.equal(-p, mhc_orthogonalize(m))


def test_autograd_sees_that_gradients_were_written_into_a_saved_tensor():
    q, f = torch.randn(1, 4, 2, 64, device="cuda"), torch.rand(32, device="cuda")
    leaf = torch.randn(2, 1, 4, 2, 64, device="cuda", requires_grad=True)
    buf = torch.zeros(2, 1, 4, 2, 64, device="cuda")
    y = (leaf * buf).sum()   # saves buf
    version = buf._version
    mhc_qk_norm_rope_backward(q, q.clone(), None, f, q.clone(), q.clone(), grad_out=(buf[0], buf[1]))
    torch.cuda.synchronize()
    assert buf._version > version
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():   # tensors without a version
        mhc_qk_norm_rope_backward(q, q.clone(), None, f, q.clone(), q.clone(),
                                  grad_out=(torch.empty_like(q), torch.empty_like(q)))


def test_orthogonalised_matrices_of_a_list_share_no_memory():
    """An operator's outputs alias nothing: one may be written, or outlive the others, alone."""
    u = [torch.randn(15, 100, device="cuda") for _ in range(70)]
    out = mhc_orthogonalize(u)
    assert len({t.untyped_storage().data_ptr() for t in out}) == len(out)
    stack = mhc_orthogonalize(torch.stack(u))
    torch.cuda.synchronize()
    assert torch.equal(torch.stack(out), stack)


def _grad_call(buf_q, buf_k, q, k, f, dq, dk):
    out = mhc_qk_norm_rope_backward(q, k, None, f, dq, dk, grad_out=(buf_q, buf_k))
    torch.cuda.synchronize()
    return out


def test_gradients_that_overlap_are_refused_and_interleaved_ones_are_not():
    B, S, d = 2, 9, 64
    g = torch.Generator(device="cuda").manual_seed(5)
    new = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()   # noqa: E731
    q, k, dq, dk, f = new(B, S, 4, d), new(B, S, 2, d), new(B, S, 4, d), new(B, S, 2, d), torch.rand(32, device="cuda")
    want = mhc_qk_norm_rope_backward(q, k, None, f, dq, dk)[:2]
    pack = new(B, S, 8, d)
    for a, b in ((pack[:, :, :4], pack[:, :, 3:5]), (pack[:, :, 2:6], pack[:, :, 2:4]),
                 (pack[:, :, 4:], pack[:, :, 5:7]), (pack[:, :, :4], pack.view(-1)[d // 2:d // 2 + B * S * 8 * d - 8 * d]
                                                     .as_strided((B, S, 2, d), pack.stride()))):
        with pytest.raises(ValueError, match="overlaps grad_out dq"):
            _grad_call(a, b, q, k, f, dq, dk)
    same = new(B, S, 4, d)
    with pytest.raises(ValueError, match="overlaps grad_out dq"):
        mhc_qk_norm_rope_backward(q, q.clone(), None, f, dq, dq.clone(), grad_out=(same, same))
    with pytest.raises(ValueError, match="overlaps itself"):
        _grad_call(torch.empty(B * S * 4 * d, dtype=torch.bfloat16, device="cuda").as_strided((B, S, 4, d), (
            S * 4 * d, 4 * d, d // 2, 1)), new(B, S, 2, d), q, k, f, dq, dk)
    other = new(B, S, 4, d)
    with pytest.raises(ValueError, match="overlaps an input"):   # the same memory in another order of axes
        _grad_call(other.view(B, 4, S, d).transpose(1, 2), new(B, S, 2, d), other, k, f, dq, dk)
    scale = torch.ones(B * S * 4 * d, device="cuda")
    with pytest.raises(ValueError, match="overlaps an input"):
        mhc_qk_norm_rope_backward(q, k, None, f, dq, dk, row_scale=scale[:B * S].view(B, S), grad_out=(
            scale.view(torch.bfloat16)[:B * S * 4 * d].view(B, S, 4, d), new(B, S, 2, d)))
    # slices between one another: by heads, by head rows, beside the inputs they belong to, the last token's too
    _grad_call(pack[:, :, :4], pack[:, :, 4:6], q, k, f, dq, dk)
    assert torch.equal(pack[:, :, :4], want[0]) and torch.equal(pack[:, :, 4:6], want[1])
    halves = new(B, S, 4, 2, d)
    halves[..., 0, :].copy_(q)
    _grad_call(halves[..., 1, :], new(B, S, 2, d), halves[..., 0, :], k, f, dq, dk)
    assert torch.equal(halves[..., 1, :], want[0]) and torch.equal(halves[..., 0, :], q)
    beside = new(B, S, 10, d)
    beside[:, :, :4].copy_(q)
    beside[:, :, 4:6].copy_(k)
    one = beside[:, :, 6:]
    _grad_call(one, new(B, S, 2, d), beside[:, :, :4], beside[:, :, 4:6], f, dq, dk)
    assert torch.equal(one, want[0]) and torch.equal(beside[:, :, :4], q) and torch.equal(beside[:, :, 4:6], k)
    # one sequence of one token: strides of axes of one element say nothing
    t = new(1, 1, 6, d)
    r = _grad_call(t[:, :, :4], t[:, :, 4:], q[:1, :1], k[:1, :1], f, dq[:1, :1], dk[:1, :1])
    assert torch.equal(r[0], want[0][:1, :1]) and torch.equal(r[1], want[1][:1, :1])


def test_overlap_of_equal_strides_is_decided_exactly():
    """Pairs of gradients at random places of one buffer against the sets of their elements; accepted calls write
    inside the buffer."""
    import random
    rng = random.Random(11)
    buf, f = torch.zeros(20000, device="cuda"), torch.rand(2, device="cuda")
    met = 0
    for _ in range(300):
        B, S, Hq, Hk, d = rng.randint(1, 3), rng.randint(1, 4), rng.randint(1, 3), rng.randint(1, 3), 4
        strides = [d * rng.randint(1, 3)]
        strides.append(strides[0] * rng.randint(1, 8) + rng.choice([0, 0, d, 3]))
        strides.append(strides[1] * rng.randint(1, 5) + rng.choice([0, 0, d, 3]))
        order = rng.choice([(2, 1, 0), (1, 2, 0), (2, 0, 1)])   # which of them batch, sequence and heads take
        st = tuple(strides[i] for i in order) + (1,)
        a = buf.as_strided((B, S, Hq, d), st, 4000)
        b = buf.as_strided((B, S, Hk, d), st, 4000 + rng.randint(-60, 60))
        places = lambda t: set((torch.arange(20000).as_strided(t.shape, st, t.storage_offset())).flatten().tolist())   # noqa: E731
        share = bool(places(a) & places(b))
        met += share
        q, k = torch.randn(B, S, Hq, d, device="cuda"), torch.randn(B, S, Hk, d, device="cuda")
        call = lambda: mhc_qk_norm_rope_backward(q, k, None, f, q.clone(), k.clone(), grad_out=(a, b))   # noqa: E731
        if share:
            with pytest.raises(ValueError, match="overlaps grad_out dq"):
                call()
        else:
            call()
    torch.cuda.synchronize()
    assert 30 < met < 270


def test_learning_rate_and_workspace_may_not_lie_in_what_is_written():
    p, g, m = (torch.randn(24, 4096, device="cuda") for _ in range(3))
    lr = torch.full((4,), 0.01, device="cuda")
    mhc_muon_step(p, g, m, lr[3:])
    mhc_muon_step(p, g, m, g.view(-1)[5:6])   # only read
    for inside in (p, m):
        before = p.clone(), m.clone()
        with pytest.raises(RuntimeError, match="overlap"):
            mhc_muon_step(p, g, m, inside.view(-1)[5:6])
        torch.cuda.synchronize()
        assert torch.equal(p, before[0]) and torch.equal(m, before[1])
    lib, vp = _lib.load(), lambda x: ctypes.cast(x, ctypes.c_void_p)
    n = ctypes.c_size_t(0)
    assert lib.mhc_ortho_workspace_size(1, 24, 4096, ctypes.byref(n)) == 0 and n.value > 0
    one = torch.zeros(24 * 4096 * 4 + n.value, dtype=torch.uint8, device="cuda")
    out = one[:24 * 4096 * 4].view(torch.float32)
    co = (ctypes.c_double * 3)(1.5, -0.5, 0.0)
    src, dst = (ctypes.c_void_p * 1)(g.data_ptr()), (ctypes.c_void_p * 1)(out.data_ptr())
    for ws, want in ((out.data_ptr() + 256, 11), (one.data_ptr() + 24 * 4096 * 4, 0)):
        a = _lib.OrthoArgs(inp=vp(src), out=vp(dst), count=1, rows=24, cols=4096, dtype=2, steps=1, coeffs=vp(co),
                           eps=1e-7, workspace=ws, workspace_bytes=n.value)
        assert lib.mhc_orthogonalize(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == want
    torch.cuda.synchronize()
