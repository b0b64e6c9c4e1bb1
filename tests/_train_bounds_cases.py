"""The cases of the operators around a training step that the debug-bounds test
runs twice, through the C ABI: in a child process on the -DMHC_DEBUG_BOUNDS
library, where the record of out-of-buffer accesses must stay empty after every
call, and in the test process on the normal library.

    python -m tests._train_bounds_cases OUT.npz     (child: writes every output)
"""
from __future__ import annotations

import ctypes
import sys

import numpy as np
import torch

from mhc_ops_b200 import _lib

# (B, S, Hq, Hk, Hv, d, rot, interleaved, dtype): vector and other kernels, partial rows of lanes, strided rows
ROPE = ((1, 1, 32, 8, 8, 128, 128, 0, torch.bfloat16), (2, 37, 5, 1, 1, 96, 32, 0, torch.float16),
        (1, 131, 3, 2, 0, 256, 64, 1, torch.bfloat16), (3, 7, 3, 1, 1, 50, 24, 1, torch.float32),
        (1, 65, 2, 1, 1, 33, 10, 0, torch.bfloat16), (1, 600, 4, 2, 2, 64, 64, 0, torch.float32))
# (count, rows, cols, dtype): one launch and three, whole vectors and not, transposed, clusters, several launches
MATS = ((1, 8, 1000, torch.float32), (3, 15, 333, torch.bfloat16), (1, 24, 5000, torch.float32), (2, 24, 4097, torch.float32),
        (2, 35, 2001, torch.bfloat16), (1, 48, 640, torch.float32), (9, 63, 500, torch.float32), (2, 80, 2052, torch.bfloat16),
        (1, 3000, 24, torch.float32), (1, 200, 80, torch.float32), (70, 3, 40, torch.float32))
DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _check_record(where: str, debug: bool) -> None:
    torch.cuda.synchronize()
    if debug:
        rec = _lib.debug_bounds(clear=True, raise_on_hit=False)
        assert rec["count"] == 0, f"{where}: access outside the call's buffers {rec}"


def _heads(t):
    return _lib.Heads() if t is None else _lib.Heads(t.data_ptr(), *t.stride()[:3])


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _rope(keep, debug):
    lib = _lib.load()
    for i, (B, S, Hq, Hk, Hv, d, rot, inter, dt) in enumerate(ROPE):
        g = torch.Generator(device="cuda").manual_seed(i)
        rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")   # noqa: E731
        x = rnd(B, S, Hq + Hk + Hv, d).to(dt)
        parts = x.split((Hq, Hk, Hv), dim=2)
        q, k, v = parts[0], parts[1], (parts[2] if Hv else None)
        ups = [rnd(*t.shape).to(dt) for t in (q, k)] + ([rnd(*v.shape).to(dt)] if Hv else [None])
        pos = (torch.arange(S, device="cuda") + 1000).expand(B, S).contiguous()
        f = torch.rand(rot // 2, generator=g, device="cuda")
        wq, wk, sc = 1 + 0.1 * rnd(d), 1 + 0.1 * rnd(d), 1 + 0.1 * rnd(B, S).abs()
        outs = [torch.zeros(t.shape, dtype=dt, device="cuda") for t in (q, k)] + (
            [torch.zeros(v.shape, dtype=dt, device="cuda")] if Hv else [None])
        a = _lib.QkArgs(q=_heads(q), k=_heads(k), v=_heads(v), q_out=_heads(outs[0]), k_out=_heads(outs[1]),
                        v_out=_heads(outs[2]), q_weight=wq.data_ptr(), k_weight=wk.data_ptr(), positions=pos.data_ptr(),
                        inv_freq=f.data_ptr(), row_scale=sc.data_ptr(), position_batch_stride=S, position_seq_stride=1,
                        batch=B, seq=S, q_heads=Hq, k_heads=Hk, v_heads=Hv, d=d, rot=rot, position_bytes=8,
                        interleaved=inter, dtype=DTYPES[dt], eps=1e-6)
        _lib.check(lib.mhc_qk_norm_rope(a, _stream()), "mhc_qk_norm_rope")
        _check_record(f"rope {i} forward", debug)
        keep(f"rope{i}/fwd", outs)
        grads = [torch.zeros_like(t) if t is not None else None for t in outs]
        dwq, dwk, dsc = torch.zeros(d, device="cuda"), torch.zeros(d, device="cuda"), torch.zeros(B, S, device="cuda")
        n = ctypes.c_size_t(0)
        _lib.check(lib.mhc_qk_norm_rope_bwd_workspace_size(B * S, d, ctypes.byref(n)), "workspace size")
        ws = torch.zeros(n.value, dtype=torch.uint8, device="cuda")
        b = _lib.QkBwdArgs(fwd=a, dq_out=_heads(ups[0]), dk_out=_heads(ups[1]), dv_out=_heads(ups[2]),
                           dq=_heads(grads[0]), dk=_heads(grads[1]), dv=_heads(grads[2]), dq_weight=dwq.data_ptr(),
                           dk_weight=dwk.data_ptr(), d_row_scale=dsc.data_ptr(), workspace=ws.data_ptr(),
                           workspace_bytes=n.value)
        _lib.check(lib.mhc_qk_norm_rope_bwd(b, _stream()), "mhc_qk_norm_rope_bwd")
        _check_record(f"rope {i} backward", debug)
        keep(f"rope{i}/bwd", grads + [dwq, dwk, dsc])
        # a workspace a byte short is refused
        b.workspace_bytes = 1
        assert lib.mhc_qk_norm_rope_bwd(b, _stream()) == 4


def _mats(keep, debug):
    lib = _lib.load()
    co = (ctypes.c_double * 15)(*((3.4445, -4.7750, 2.0315) * 5))
    ptrs = lambda t: (ctypes.c_void_p * t.shape[0])(*[x.data_ptr() for x in t])   # noqa: E731
    vp = lambda a: ctypes.cast(a, ctypes.c_void_p)   # noqa: E731
    for i, (L, R, C, dt) in enumerate(MATS):
        g = torch.Generator(device="cuda").manual_seed(50 + i)
        u = (torch.randn(L, R, C, generator=g, device="cuda") * 1e-3).to(dt)
        out = torch.zeros_like(u)
        n = ctypes.c_size_t(0)
        _lib.check(lib.mhc_ortho_workspace_size(L, R, C, ctypes.byref(n)), "workspace size")
        ws = torch.zeros(max(n.value, 256), dtype=torch.uint8, device="cuda")
        keep_alive = [ptrs(u), ptrs(out)]
        a = _lib.OrthoArgs(inp=vp(keep_alive[0]), out=vp(keep_alive[1]), count=L, rows=R, cols=C, dtype=DTYPES[dt],
                           steps=5, coeffs=vp(co), eps=1e-7, workspace=ws.data_ptr(), workspace_bytes=n.value)
        _lib.check(lib.mhc_orthogonalize(a, _stream()), "mhc_orthogonalize")
        _check_record(f"matrices {i} orthogonalize", debug)
        keep(f"mats{i}/ortho", [out])
        if n.value:
            a.workspace_bytes = n.value - 1
            assert lib.mhc_orthogonalize(a, _stream()) == 4
            a.workspace_bytes = n.value
        # in place
        v = u.clone()
        inp = ptrs(v)
        a.inp = a.out = vp(inp)
        _lib.check(lib.mhc_orthogonalize(a, _stream()), "mhc_orthogonalize in place")
        _check_record(f"matrices {i} in place", debug)
        assert torch.equal(v, out)
        p = (torch.randn(L, R, C, generator=g, device="cuda")).to(dt)
        m = torch.randn(L, R, C, generator=g, device="cuda") * 1e-3
        lr = torch.full((1,), 0.1, device="cuda")
        pp, gg, mm = ptrs(p), ptrs(u), ptrs(m)
        s = _lib.MuonArgs(params=vp(pp), grads=vp(gg), momenta=vp(mm), count=L, rows=R, cols=C, param_dtype=DTYPES[dt],
                          grad_dtype=DTYPES[dt], nesterov=1, steps=5, coeffs=vp(co), eps=1e-7, momentum=0.9,
                          weight_decay=0.1, scale=1.0, lr=0.0, lr_device=lr.data_ptr(), workspace=ws.data_ptr(),
                          workspace_bytes=n.value)
        _lib.check(lib.mhc_muon_step(s, _stream()), "mhc_muon_step")
        _check_record(f"matrices {i} update", debug)
        keep(f"mats{i}/muon", [p, m])


def run_cases(debug: bool) -> dict[str, np.ndarray]:
    out: dict[str, np.ndarray] = {}

    def keep(tag, tensors):
        for i, t in enumerate(tensors):
            if t is not None:
                t = t.detach().contiguous().cpu()
                out[f"{tag}/{i}"] = (t if t.dtype == torch.float32 else t.view(torch.uint8)).numpy().copy()

    _rope(keep, debug)
    _mats(keep, debug)
    return out


if __name__ == "__main__":
    _lib.debug_bounds(clear=True)
    np.savez(sys.argv[1], **run_cases(debug=True))
