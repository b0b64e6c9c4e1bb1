"""The mHC pre-op as registered torch operators: ``torch.ops.mhc.fwd`` and
``torch.ops.mhc.bwd`` (``TORCH_LIBRARY(mhc, ...)`` in ``csrc/torch_ops.cpp``).

``fwd(x, phi, alpha, bias, norm_eps=1e-6, hc_eps=1e-6)`` returns
``(h_in, h_post, h_res, inv_rms, h_mix, h_pre)``: the reference's
``mhc_forward_pre(..., outflag=True)`` (``src/forward/golden.py:10-69``),
whose Triton call site is ``src/forward/mhc_forward_pre_triton.py:409-417``.

``bwd(x, phi, alpha, inv_rms, h_mix, h_pre, h_post, dh_in, dh_post, dh_res,
gamma, norm_eps=1e-6, hc_eps=1e-6)`` returns ``(dx, dphi, dalpha, dbias,
dgamma)``: the reference's ``mhc_backward_manual``
(``src/backward/golden.py:10-96``), Triton call site
``src/backward/mhc_backward_triton.py:467-473``; ``gamma`` may be None.

``qk_norm_rope`` / ``qk_norm_rope_bwd`` / ``qk_norm_rope_bwd_into``,
``orthogonalize`` and ``muon_step_`` are the operators under
``mhc_qk_norm_rope``, ``mhc_orthogonalize`` and ``mhc_muon_step``
(``mhc_ops_b200.qkrope``, ``mhc_ops_b200.muon``), which document them.  A
backward pass through one of their results, and a forward-mode tangent on an
input, raises: the differentiable forms are the autograd Functions of
``mhc_ops_b200.qkrope``.

The operators run the same kernels as the ctypes API through the C ABI, on the
current CUDA stream, and have Meta kernels, so FakeTensor tracing
(``torch.compile``, ``torch.export``) sees them as single graph nodes.  CPU
tensors fail (there is no CPU kernel).  ``check_status()`` waits for the
device status copies of the operators' workspaces and raises if a kernel's
bounded wait expired in an earlier call.
"""
from __future__ import annotations

import os
import threading

import torch

_LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib", "libmhc_torch.so")
_lock = threading.Lock()
_loaded = False

__all__ = ["load", "fwd", "bwd", "qk_norm_rope", "qk_norm_rope_bwd", "qk_norm_rope_bwd_into", "orthogonalize",
           "muon_step_", "check_status", "lib_path"]


def lib_path() -> str:
    return _LIB_PATH


def load() -> None:
    """Register the ``mhc`` operators (once); raises if the library is not built.  Call it before a program whose
    first use of them is inside ``torch.compile``, which cannot trace the loading."""
    global _loaded
    if _loaded:
        return
    with _lock:
        if not _loaded:
            if not os.path.exists(_LIB_PATH):
                raise RuntimeError(f"libmhc_torch.so not found at {_LIB_PATH}; build it with "
                                   "`python -m mhc_ops_b200.build` (there is no fallback)")
            torch.ops.load_library(_LIB_PATH)
            for name in _BOUND:
                globals()[name] = getattr(torch.ops.mhc, name).default
            _loaded = True


def fwd(x, phi, alpha, bias, norm_eps: float = 1e-6, hc_eps: float = 1e-6):
    load()
    return torch.ops.mhc.fwd(x, phi, alpha, bias, norm_eps, hc_eps)


def bwd(x, phi, alpha, inv_rms, h_mix, h_pre, h_post, dh_in, dh_post, dh_res, gamma=None,
        norm_eps: float = 1e-6, hc_eps: float = 1e-6):
    load()
    return torch.ops.mhc.bwd(x, phi, alpha, inv_rms, h_mix, h_pre, h_post, dh_in, dh_post, dh_res, gamma,
                             norm_eps, hc_eps)


# The operators' calls without the overload lookup; load() puts them in place of these, which serve a first call.
_BOUND = ("qk_norm_rope", "qk_norm_rope_bwd", "qk_norm_rope_bwd_into", "orthogonalize", "muon_step_")


def qk_norm_rope(*args):
    load()
    return torch.ops.mhc.qk_norm_rope.default(*args)


def qk_norm_rope_bwd(*args):
    load()
    return torch.ops.mhc.qk_norm_rope_bwd.default(*args)


def qk_norm_rope_bwd_into(*args):
    load()
    return torch.ops.mhc.qk_norm_rope_bwd_into.default(*args)


def orthogonalize(*args):
    load()
    return torch.ops.mhc.orthogonalize.default(*args)


def muon_step_(*args):
    load()
    return torch.ops.mhc.muon_step_.default(*args)


def untracked(out):
    """An operator's results without the node that refuses a gradient: the functions that are no autograd Functions
    return plain tensors whatever their inputs require, as ``mhc_forward_pre`` does."""
    return [t.detach() for t in out] if out[0].requires_grad else out


def check_status() -> None:
    load()
    torch.ops.mhc.check_status()
