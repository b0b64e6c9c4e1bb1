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
phi at n = 8.  All sums run in 64 bits (32 would lose small singular values,
which the steps lift a few hundred times) and the result is rounded once.  The
reference has no optimiser.
"""
from __future__ import annotations

import torch

from . import ops

__all__ = ["NEWTON_SCHULZ_COEFFS", "mhc_orthogonalize", "mhc_muon_step"]

# The usual quintic: it lifts small singular values 3.4445-fold a step and
# leaves the others in about [0.7, 1.2].
NEWTON_SCHULZ_COEFFS = ((3.4445, -4.7750, 2.0315),) * 5


def _list(x, name):
    """A tensor as a list of one (the operators take a stack as such), a sequence as it is."""
    x = [x] if torch.is_tensor(x) else list(x)
    if not x:
        raise ValueError(f"{name} must not be an empty sequence")
    if not torch.is_tensor(x[0]):
        raise ValueError(f"{name} must be a tensor or a sequence of tensors")
    if x[0].device.type == "cpu":
        raise RuntimeError(f"mhc_ops_b200 runs on CUDA only: {name} is on the CPU (there is no CPU fallback)")
    return x


def _coeffs(coeffs):
    steps = [tuple(step) for step in coeffs]   # once: coeffs may be a generator
    if any(len(step) != 3 for step in steps):
        raise ValueError("coeffs must be 1 to 16 triples (a, b, c)")
    return [c for step in steps for c in step]


def mhc_orthogonalize(g, coeffs=NEWTON_SCHULZ_COEFFS, eps: float = 1e-7):
    """Orthogonalise a matrix ``[rows, cols]``, a stack ``[count, rows, cols]`` or a sequence of
    equal matrices, fp32 or bf16, with ``min(rows, cols) <= 80``.

    Returns the same kind (a list for a sequence) in the input's type.  Every
    matrix is treated alone; repeated calls return the same bits.  Records no gradient.
    """
    out = ops.untracked(ops.orthogonalize(_list(g, "g"), _coeffs(coeffs), eps))
    return out[0] if torch.is_tensor(g) else out


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
    lr_tensor = None
    if torch.is_tensor(lr):
        if lr.is_cuda:
            lr_tensor, lr = lr, 0.0
        else:
            lr = lr.item()
    ops.muon_step_(_list(params, "params"), _list(grads, "grads"), _list(momenta, "momenta"), lr_tensor, lr, momentum,
                   nesterov, weight_decay, scale, _coeffs(coeffs), eps)
