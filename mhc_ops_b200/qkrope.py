"""Norms of queries and keys for each head, with the rotary position rotation in the same pass.

What stands between the projection of ``h_in`` and the attention of a
hyper-connection block's sublayer.  For every head row ``x [d]`` of a token at
position ``p``, with ``s`` the token's row factor (1 without ``row_scale``)::

    z = s x,   a = z * w / sqrt(mean(z^2) + eps),   y = a turned by the angles p * inv_freq
    v_out = s v

``row_scale`` takes the ``h_in_rstd`` that ``mhc_forward_pre_fused_norm``
returns: with the weight of the sublayer's RMSNorm folded into the projection's
columns, the projection runs on ``h_in`` itself, ``RMSNorm(h_in)`` is never
written, and this pass applies the factor to q, k and v.

The reference stops at ``h_in`` (``src/forward/golden.py:62-63``).  bf16, fp16
or fp32 tensors (sums in fp32), any strides with unit stride along ``d``; CPU
tensors raise.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import ops

__all__ = ["mhc_qk_norm_rope", "mhc_qk_norm_rope_backward", "MHCQKNormRopeFunction", "mhc_qk_norm_rope_fn",
           "MHCQKVNormRopeFunction", "mhc_qkv_norm_rope_fn"]


def _check(q):
    if not torch.is_tensor(q):
        raise ValueError("q must be a tensor of shape [B, S, heads, d]")
    if q.device.type == "cpu":
        raise RuntimeError("mhc_ops_b200 runs on CUDA only: q is on the CPU (there is no CPU fallback)")


def mhc_qk_norm_rope(q, k, positions, inv_freq, q_weight=None, k_weight=None, *, v=None, row_scale=None,
                     eps: float = 1e-6, interleaved: bool = False):
    """RMSNorm of every query and key head row, then its rotary rotation, in one pass.

    ``q [B,S,Hq,d]``, ``k [B,S,Hk,d]`` and the optional ``v [B,S,Hv,d]`` may be
    views of one packed projection.  ``positions`` are int32/int64 ``[B,S]`` or
    ``[S]`` (None: 0 .. S-1), of any value below 2^31 in magnitude;
    ``inv_freq [rot/2]``, taken in fp32, the angles per position of the
    ``rot <= d`` leading elements that turn, in pairs ``(i, i + rot/2)`` or, ``interleaved``,
    ``(2i, 2i + 1)``.  ``q_weight`` / ``k_weight [d]`` are the norms' weights
    (None: ones), ``row_scale [B,S]`` the factor every head of a token is
    multiplied with first.  ``d`` is 1 to 1024.  Returns contiguous ``(q_out,
    k_out)``, with ``v`` also ``v_out = row_scale * v``.  Records no gradient:
    ``mhc_qk_norm_rope_fn`` and ``mhc_qkv_norm_rope_fn`` do.
    """
    _check(q)
    return tuple(ops.untracked(ops.qk_norm_rope(q, k, positions, inv_freq, q_weight, k_weight, v, row_scale, eps,
                                                interleaved)))


def mhc_qk_norm_rope_backward(q, k, positions, inv_freq, dq_out, dk_out, q_weight=None, k_weight=None, *, v=None,
                              dv_out=None, row_scale=None, eps: float = 1e-6, interleaved: bool = False,
                              grad_out=None, weight_grads: bool = True, row_scale_grad: bool = True):
    """Gradients of ``mhc_qk_norm_rope`` from the upstream ``dq_out``, ``dk_out`` (and ``dv_out`` with ``v``).

    Returns ``(dq, dk, dv, dq_weight, dk_weight, drow_scale)``; an entry whose
    input is None, or that ``weight_grads`` / ``row_scale_grad`` switch off, is
    None.  Weight and row factor gradients are fp32; repeated calls return the
    same bits.  ``grad_out`` is an optional ``(dq, dk)`` or ``(dq, dk, dv)`` of
    tensors the gradients are written into, for instance the three slices of
    the packed gradient that the projection's backward takes; they must not
    overlap the inputs, each other or themselves.  Slices of one tensor may lie
    between one another; a tensor of other strides than an input's has to lie
    wholly apart from it.
    """
    _check(q)
    args = (q, k, positions, inv_freq, dq_out, dk_out, q_weight, k_weight, v, dv_out, row_scale, eps, interleaved,
            weight_grads, row_scale_grad)
    count = 2 if v is None else 3
    if grad_out is None:
        out = ops.untracked(ops.qk_norm_rope_bwd(*args))
        grads, rest = out[:count], out[count:]
    elif torch.compiler.is_compiling():
        # a traced operator that writes into given tensors may not return others: one copy more
        out = ops.untracked(ops.qk_norm_rope_bwd(*args))
        grads, rest = list(grad_out), out[count:]
        if len(grads) != count:
            raise ValueError(f"grad_out must hold {count} tensors")
        for t, g in zip(grads, out):
            t.copy_(g)
    else:
        grads = list(grad_out)
        rest = ops.qk_norm_rope_bwd_into(*args, grads)
    rest = iter(rest)
    dwq = next(rest) if q_weight is not None and weight_grads else None
    dwk = next(rest) if k_weight is not None and weight_grads else None
    dsc = next(rest) if row_scale is not None and row_scale_grad else None
    return grads[0], grads[1], None if v is None else grads[2], dwq, dwk, dsc


def _cast(g, like):
    return None if g is None else g.to(like.dtype)


class MHCQKNormRopeFunction(torch.autograd.Function):
    """autograd over ``mhc_qk_norm_rope``: gradients for q, k, v, the weights and row_scale."""

    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, q_weight, k_weight, v, row_scale, eps, interleaved):
        ctx.save_for_backward(q, k, positions, inv_freq, q_weight, k_weight, v, row_scale)
        ctx.opts = (eps, interleaved)
        return mhc_qk_norm_rope(q, k, positions, inv_freq, q_weight, k_weight, v=v, row_scale=row_scale, eps=eps,
                                interleaved=interleaved)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq_out, dk_out, dv_out=None):
        q, k, positions, inv_freq, q_weight, k_weight, v, row_scale = ctx.saved_tensors
        need = ctx.needs_input_grad
        dq, dk, dv, dwq, dwk, dsc = mhc_qk_norm_rope_backward(
            q, k, positions, inv_freq, dq_out, dk_out, q_weight, k_weight, v=v, dv_out=dv_out, row_scale=row_scale,
            eps=ctx.opts[0], interleaved=ctx.opts[1], weight_grads=need[4] or need[5], row_scale_grad=need[7])
        return dq, dk, None, None, _cast(dwq, q_weight), _cast(dwk, k_weight), dv, _cast(dsc, row_scale), None, None


class MHCQKVNormRopeFunction(torch.autograd.Function):
    """The same on one packed projection ``qkv [B,S,Hq+2Hk,d]``, whose gradient
    is written as one packed tensor (no concatenation)."""

    @staticmethod
    def forward(ctx, qkv, q_heads, k_heads, positions, inv_freq, q_weight, k_weight, row_scale, eps, interleaved):
        if not torch.is_tensor(qkv) or qkv.dim() != 4 or qkv.shape[2] != q_heads + 2 * k_heads:
            raise ValueError(f"qkv must be a tensor of shape [B, S, {q_heads + 2 * k_heads}, d]")
        ctx.save_for_backward(qkv, positions, inv_freq, q_weight, k_weight, row_scale)
        ctx.opts = (q_heads, k_heads, eps, interleaved)
        q, k, v = qkv.split((q_heads, k_heads, k_heads), dim=2)
        return mhc_qk_norm_rope(q, k, positions, inv_freq, q_weight, k_weight, v=v, row_scale=row_scale, eps=eps,
                                interleaved=interleaved)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq_out, dk_out, dv_out):
        qkv, positions, inv_freq, q_weight, k_weight, row_scale = ctx.saved_tensors
        q_heads, k_heads, eps, interleaved = ctx.opts
        need = ctx.needs_input_grad
        parts = (q_heads, k_heads, k_heads)
        q, k, v = qkv.split(parts, dim=2)
        dqkv = torch.empty(qkv.shape, dtype=qkv.dtype, device=qkv.device)
        _, _, _, dwq, dwk, dsc = mhc_qk_norm_rope_backward(
            q, k, positions, inv_freq, dq_out, dk_out, q_weight, k_weight, v=v, dv_out=dv_out, row_scale=row_scale,
            eps=eps, interleaved=interleaved, grad_out=dqkv.split(parts, dim=2), weight_grads=need[5] or need[6],
            row_scale_grad=need[7])
        return (dqkv, None, None, None, None, _cast(dwq, q_weight), _cast(dwk, k_weight), _cast(dsc, row_scale), None,
                None)


def _other(t, u):
    """``t``, as a view where it is ``u`` itself: ``torch.compile`` keeps one of the gradients of a tensor that an
    autograd Function takes twice."""
    return t.view_as(t) if t is not None and t is u else t


def mhc_qk_norm_rope_fn(q, k, positions, inv_freq, q_weight=None, k_weight=None, *, v=None, row_scale=None,
                        eps: float = 1e-6, interleaved: bool = False):
    """Differentiable ``mhc_qk_norm_rope``."""
    k, v, k_weight = _other(k, q), _other(_other(v, q), k), _other(k_weight, q_weight)
    return MHCQKNormRopeFunction.apply(q, k, positions, inv_freq, q_weight, k_weight, v, row_scale, eps, interleaved)


def mhc_qkv_norm_rope_fn(qkv, q_heads: int, k_heads: int, positions, inv_freq, q_weight=None, k_weight=None, *,
                         row_scale=None, eps: float = 1e-6, interleaved: bool = False):
    """Differentiable ``mhc_qk_norm_rope`` on a packed projection ``[B,S,Hq+2Hk,d]``: returns ``(q, k, v)``."""
    k_weight = _other(k_weight, q_weight)
    return MHCQKVNormRopeFunction.apply(qkv, q_heads, k_heads, positions, inv_freq, q_weight, k_weight, row_scale,
                                        eps, interleaved)
