"""Host side of the operators around a training step, without a GPU: struct
mirrors, device-free answers of the C entry points, refusal of CPU tensors,
and the data-parallel update's bookkeeping with an injected update."""
import ctypes
import os
import subprocess
import tempfile

import pytest
import torch

from mhc_ops_b200 import (_lib, mhc_muon_step, mhc_orthogonalize, mhc_qk_norm_rope, mhc_qk_norm_rope_backward)
from mhc_ops_b200.backward import param_grad_numel
from mhc_ops_b200.dist import DataParallelMHC

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    from mhc_ops_b200 import build
    build.build()
    return _lib.load()


def test_ctypes_structs_match_c_layout():
    classes = {"mhc_heads": _lib.Heads, "mhc_qk_args": _lib.QkArgs, "mhc_qk_bwd_args": _lib.QkBwdArgs,
               "mhc_ortho_args": _lib.OrthoArgs, "mhc_muon_args": _lib.MuonArgs}
    lines = []
    for s, cls in classes.items():
        lines.append(f'printf("{s} %zu\\n", sizeof({s}));')
        for f, _ in cls._fields_:
            c = "in" if f == "inp" else f
            lines.append(f'printf("{s}.{f} %zu\\n", offsetof({s}, {c}));')
    src = ('#include <stdio.h>\n#include <stddef.h>\n#include "mhc_ops.h"\nint main(void) {\n' + "\n".join(lines)
           + "\nreturn 0; }\n")
    with tempfile.TemporaryDirectory() as d:
        c, exe = os.path.join(d, "layout.c"), os.path.join(d, "layout")
        open(c, "w").write(src)
        subprocess.run(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), c, "-o", exe], check=True)
        out = subprocess.run([exe], capture_output=True, text=True, check=True).stdout
    for line in out.split("\n"):
        if not line.strip():
            continue
        key, val = line.split()
        if "." in key:
            s, f = key.split(".")
            assert getattr(classes[s], f).offset == int(val), key
        else:
            assert ctypes.sizeof(classes[key]) == int(val), key


def test_entry_points_answer_without_a_device(lib):
    BAD, NULL = 2, 1
    for fn in (lib.mhc_qk_norm_rope, lib.mhc_qk_norm_rope_bwd, lib.mhc_orthogonalize, lib.mhc_muon_step):
        assert fn(None, None) == NULL
    ok = dict(batch=1, seq=1, q_heads=1, k_heads=1, d=64, rot=64, eps=1e-6)
    for bad in (dict(batch=-1), dict(seq=-1), dict(q_heads=0), dict(k_heads=0), dict(v_heads=-1), dict(d=0),
                dict(d=1025, rot=0), dict(rot=63), dict(rot=66), dict(rot=-2), dict(dtype=3), dict(dtype=-1),
                dict(eps=-1.0), dict(eps=float("nan")), dict(batch=1 << 20, seq=1 << 20),
                dict(positions=16, position_bytes=2)):
        a = _lib.QkArgs(**{**ok, **bad})
        assert lib.mhc_qk_norm_rope(a, None) == BAD, bad
        assert lib.mhc_qk_norm_rope_bwd(_lib.QkBwdArgs(fwd=a), None) == BAD, bad
    co = (ctypes.c_double * 3)(1.5, -0.5, 0.0)
    ok = dict(count=1, rows=8, cols=64, steps=1, eps=1e-7, coeffs=ctypes.cast(co, ctypes.c_void_p))
    for bad, want in ((dict(rows=81, cols=81), BAD), (dict(count=-1), BAD), (dict(rows=-1), BAD), (dict(steps=0), BAD),
                      (dict(steps=17), BAD), (dict(eps=0.0), BAD), (dict(eps=float("nan")), BAD),
                      (dict(coeffs=None), NULL), (dict(cols=(1 << 30) + 1), BAD)):
        assert lib.mhc_orthogonalize(_lib.OrthoArgs(**{**ok, **bad, "dtype": 2}), None) == want, bad
        assert lib.mhc_muon_step(_lib.MuonArgs(**{**ok, **bad, "param_dtype": 2, "grad_dtype": 2}), None) == want, bad
    assert lib.mhc_orthogonalize(_lib.OrthoArgs(**ok, dtype=1), None) == BAD
    assert lib.mhc_muon_step(_lib.MuonArgs(**ok, param_dtype=2, grad_dtype=1), None) == BAD
    out = ctypes.c_size_t(0)
    assert lib.mhc_ortho_workspace_size(1, 81, 81, ctypes.byref(out)) == BAD
    assert lib.mhc_ortho_workspace_size(1, 8, 64, None) == NULL
    assert lib.mhc_qk_norm_rope_bwd_workspace_size(-1, 64, ctypes.byref(out)) == BAD
    assert lib.mhc_status_string(11) != b"unknown mhc status"


def test_cpu_tensors_raise_no_fallback():
    q, k, f = torch.zeros(1, 2, 2, 8), torch.zeros(1, 2, 1, 8), torch.ones(4)
    with pytest.raises(RuntimeError, match="CUDA only"):
        mhc_qk_norm_rope(q, k, None, f)
    with pytest.raises(RuntimeError, match="CUDA only"):
        mhc_qk_norm_rope_backward(q, k, None, f, q, k)
    m = torch.zeros(3, 8)
    with pytest.raises(RuntimeError, match="CUDA only"):
        mhc_orthogonalize(m)
    with pytest.raises(RuntimeError, match="CUDA only"):
        mhc_muon_step(m, m.clone(), m.clone(), 0.1)


def test_data_parallel_update_takes_the_reduced_dphi():
    n, D = 2, 4
    calls = []

    class Pending:
        def wait(self):
            calls.append("wait")

    def update(phi, g, m, lr, **kw):
        calls.append((tuple(g.shape), float(g.sum()), lr, kw))

    dp = DataParallelMHC(n, D, fwd=lambda *a: None, bwd=lambda *a: None, muon=update)
    phi = torch.zeros(n * n + 2 * n, n * D)
    with pytest.raises(RuntimeError, match="backward"):
        dp.muon_step(phi, phi.clone(), 0.1)
    flat = dp.grad_buffer("cpu")
    assert flat.numel() == param_grad_numel(n, D)
    flat.zero_()
    flat[:phi.numel()] = 1.0
    dp.pending = Pending()
    dp.muon_step(phi, phi.clone(), 0.1, weight_decay=0.5)
    assert calls == ["wait", ((8, 8), 64.0, 0.1, {"weight_decay": 0.5})] and dp.pending is None
    with pytest.raises(ValueError, match="phi must be"):
        dp.muon_step(phi[:4], phi, 0.1)


def test_meta_kernels_give_the_output_shapes():
    """FakeTensor tracing sees each operator as one node with these outputs."""
    from mhc_ops_b200 import ops
    m = dict(device="meta", dtype=torch.bfloat16)
    q, k, v = torch.empty(2, 5, 4, 16, **m), torch.empty(2, 5, 2, 16, **m), torch.empty(2, 5, 2, 16, **m)
    f, w, s = torch.empty(8, device="meta"), torch.empty(16, device="meta"), torch.empty(2, 5, device="meta")
    out = ops.qk_norm_rope(q, k, None, f, w, None, v, s, 1e-6, False)
    assert [tuple(o.shape) for o in out] == [(2, 5, 4, 16), (2, 5, 2, 16), (2, 5, 2, 16)]
    args = (q, k, None, f, q, k, w, w, v, v, s, 1e-6, False)
    out = ops.qk_norm_rope_bwd(*args, True, True)
    assert [tuple(o.shape) for o in out] == [(2, 5, 4, 16), (2, 5, 2, 16), (2, 5, 2, 16), (16,), (16,), (2, 5)]
    assert [o.dtype for o in out[3:]] == [torch.float32] * 3
    assert [tuple(o.shape) for o in ops.qk_norm_rope_bwd_into(*args, False, True, [q, k, v])] == [(2, 5)]
    g = torch.empty(3, 8, 64, device="meta")
    assert [tuple(o.shape) for o in ops.orthogonalize([g], [1.5, -0.5, 0.0], 1e-7)] == [(3, 8, 64)]
    assert ops.muon_step_([g], [g], [g], None, 0.1, 0.9, True, 0.0, 1.0, [1.5, -0.5, 0.0], 1e-7) is None
