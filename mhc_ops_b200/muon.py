"""Updates of phi: Newton-Schulz orthogonalisation and the momentum update around it.

``mhc_backward_manual`` ends with ``dphi``; this module turns it into the next
``phi``.  ``mhc_orthogonalize`` replaces a matrix ``U`` by one with (nearly)
the same singular vectors and singular values near one::

    X = U / (|U|_F + eps);   per (a, b, c) of coeffs:  X <- a X + (b A + c A^2) X,  A = X X^T

and ``mhc_muon_step`` applies the whole update in place, for the phi of every
layer in one call::

    m <- mu m + (1 - mu) g;   u = mu m + (1 - mu) g  (nesterov)  or  m
    phi <- (1 - lr weight_decay) phi - lr scale orthogonalised(u)

The shorter side of a matrix may have up to 80 rows, the ``n*n + 2n`` rows of
phi at n = 8.  Sums over the long side and the iteration run in 64 bits, the
last product in 32.  The reference has no optimiser.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib

__all__ = ["NEWTON_SCHULZ_COEFFS", "mhc_orthogonalize", "mhc_muon_step"]

# The usual quintic: it lifts small singular values 3.4445-fold a step and
# leaves the others in about [0.7, 1.2].
NEWTON_SCHULZ_COEFFS = ((3.4445, -4.7750, 2.0315),) * 5

_TYPES = (torch.float32, torch.bfloat16)


class _Mats:
    """Equal matrices as the C ABI takes them: a host array of pointers and what they share."""

    def __init__(self, x, name, copy):
        """``x``: a [rows, cols] or [count, rows, cols] tensor, or a sequence of [rows, cols] tensors.
        ``copy``: make non-contiguous ones contiguous instead of refusing them."""
        if torch.is_tensor(x):
            if x.dim() not in (2, 3):
                raise ValueError(f"{name} must be [rows, cols] or [count, rows, cols], got {tuple(x.shape)}")
            if not x.is_contiguous():
                if not copy:
                    raise ValueError(f"{name} must be contiguous")
                x = x.contiguous()
            self.keep = x
            self.shape = tuple(x.shape[-2:])
            self.count = 1 if x.dim() == 2 else x.shape[0]
            base, step = x.data_ptr(), self.shape[0] * self.shape[1] * x.element_size()
            ptrs = [base + i * step for i in range(self.count)]
            first = x
        else:
            x = list(x)
            if not x:
                raise ValueError(f"{name} must not be an empty sequence")
            first = x[0]
            if not torch.is_tensor(first) or first.dim() != 2:
                raise ValueError(f"{name} must hold [rows, cols] tensors")
            shape, dtype, dev = first.shape, first.dtype, first.device
            for i, t in enumerate(x):
                if t.shape != shape or t.dtype != dtype or t.device != dev:
                    raise ValueError(f"{name}[{i}] is {t.dtype} {tuple(t.shape)} on {t.device}, {name}[0] is {dtype} "
                                     f"{tuple(shape)} on {dev}")
                if not t.is_contiguous():
                    if not copy:
                        raise ValueError(f"{name}[{i}] must be contiguous")
                    x[i] = t.contiguous()
            self.keep = x
            self.shape = tuple(shape)
            self.count = len(x)
            ptrs = [t.data_ptr() for t in x]
        if not first.is_cuda:
            raise RuntimeError(f"mhc_ops_b200 runs on CUDA only: {name} is on the CPU (there is no CPU fallback)")
        if first.dtype not in _TYPES:
            raise TypeError(f"{name} must be float32 or bfloat16, got {first.dtype}")
        if min(self.shape) > 80:
            raise ValueError(f"{name} is {self.shape[0]} x {self.shape[1]}: the shorter side may have at most 80 rows")
        self.dtype, self.device = first.dtype, first.device
        self.array = (ctypes.c_void_p * self.count)(*ptrs)
        self.ptr = ctypes.cast(self.array, ctypes.c_void_p)


def _coeffs(coeffs):
    flat = [float(c) for step in coeffs for c in step]
    if not 1 <= len(coeffs) <= 16 or len(flat) != 3 * len(coeffs):
        raise ValueError("coeffs must be 1 to 16 triples (a, b, c)")
    return (ctypes.c_double * len(flat))(*flat), len(coeffs)


def _check_eps(eps):
    if not eps >= 1e-20:
        raise ValueError(f"eps must be at least 1e-20, got {eps}")


def _workspace(lib, mats):
    nbytes = ctypes.c_size_t(0)
    _lib.check(lib.mhc_ortho_workspace_size(mats.count, *mats.shape, ctypes.byref(nbytes)), "mhc_ortho_workspace_size")
    return _lib.scratch(nbytes.value, mats.device), nbytes.value


def mhc_orthogonalize(g, coeffs=NEWTON_SCHULZ_COEFFS, eps: float = 1e-7):
    """Orthogonalise a matrix ``[rows, cols]``, a stack ``[count, rows, cols]`` or a sequence of
    equal matrices, fp32 or bf16, with ``min(rows, cols) <= 80``.

    Returns the same kind (a list for a sequence) in the input's type.  Every
    matrix is treated alone: the result does not depend on its neighbours.
    """
    _check_eps(eps)
    co, steps = _coeffs(coeffs)
    mats = _Mats(g, "g", copy=True)
    shape = g.shape if torch.is_tensor(g) else (mats.count, *mats.shape)
    out = torch.empty(shape, dtype=mats.dtype, device=mats.device)
    dst = _Mats(out, "out", copy=False)
    with torch.cuda.device(mats.device):
        lib = _lib.load()
        ws, nbytes = _workspace(lib, mats)
        args = _lib.OrthoArgs(inp=mats.ptr, out=dst.ptr, count=mats.count, rows=mats.shape[0], cols=mats.shape[1],
                              dtype=_lib.DTYPES[mats.dtype], steps=steps, coeffs=ctypes.cast(co, ctypes.c_void_p),
                              eps=float(eps), workspace=ws.data_ptr(), workspace_bytes=nbytes)
        _lib.check(lib.mhc_orthogonalize(args, torch.cuda.current_stream(mats.device).cuda_stream),
                   "mhc_orthogonalize")
    return out if torch.is_tensor(g) else list(out.unbind(0))


def mhc_muon_step(params, grads, momenta, lr, momentum: float = 0.95, nesterov: bool = True,
                  weight_decay: float = 0.0, scale: float = 1.0, coeffs=NEWTON_SCHULZ_COEFFS, eps: float = 1e-7):
    """The momentum update with an orthogonalised direction, in place on ``params`` and ``momenta``.

    ``params``, ``grads`` and ``momenta`` are each a matrix, a stack or a
    sequence of equal matrices, as many of one as of the others: parameters and
    gradients fp32 or bf16, momenta fp32 (zeros before the first step).  ``lr``
    is a number or a one-element fp32 tensor on the same device, which is read
    when the kernels run: a captured step follows a schedule written into it.
    ``scale`` multiplies the orthogonalised direction, e.g.
    ``0.2 * max(rows, cols) ** 0.5`` to match the usual size of an Adam update.
    A bf16 parameter is rounded to nearest once, after the update in fp32.
    Parameters and momenta must not overlap anything else in the call.
    """
    _check_eps(eps)
    co, steps = _coeffs(coeffs)
    p = _Mats(params, "params", copy=False)
    g = _Mats(grads, "grads", copy=True)
    m = _Mats(momenta, "momenta", copy=False)
    if not (p.count == g.count == m.count and p.shape == g.shape == m.shape):
        raise ValueError(f"params, grads and momenta differ: {p.count} of {p.shape}, {g.count} of {g.shape}, "
                         f"{m.count} of {m.shape}")
    if not (p.device == g.device == m.device):
        raise ValueError(f"params are on {p.device}, grads on {g.device}, momenta on {m.device}")
    if m.dtype != torch.float32:
        raise TypeError(f"momenta must be float32, got {m.dtype}")
    lr_dev = None
    if torch.is_tensor(lr):
        if lr.is_cuda:
            if lr.numel() != 1 or lr.dtype != torch.float32 or lr.device != p.device:
                raise ValueError(f"lr must be a number or a one-element float32 tensor on {p.device}")
            lr_dev, lr = lr, 0.0
        else:
            lr = lr.item()
    with torch.cuda.device(p.device):
        lib = _lib.load()
        ws, nbytes = _workspace(lib, p)
        args = _lib.MuonArgs(params=p.ptr, grads=g.ptr, momenta=m.ptr, count=p.count, rows=p.shape[0], cols=p.shape[1],
                             param_dtype=_lib.DTYPES[p.dtype], grad_dtype=_lib.DTYPES[g.dtype],
                             nesterov=1 if nesterov else 0, steps=steps, coeffs=ctypes.cast(co, ctypes.c_void_p),
                             eps=float(eps), momentum=float(momentum), weight_decay=float(weight_decay),
                             scale=float(scale), lr=float(lr), lr_device=_lib.ptr(lr_dev), workspace=ws.data_ptr(),
                             workspace_bytes=nbytes)
        _lib.check(lib.mhc_muon_step(args, torch.cuda.current_stream(p.device).cuda_stream), "mhc_muon_step")
    # autograd has to see that these were written
    torch.autograd.graph.increment_version([t for x in (p.keep, m.keep) for t in (x if isinstance(x, list) else [x])])
