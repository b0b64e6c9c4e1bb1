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

import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .forward import _as_f32

__all__ = ["mhc_qk_norm_rope", "mhc_qk_norm_rope_backward", "MHCQKNormRopeFunction", "mhc_qk_norm_rope_fn",
           "MHCQKVNormRopeFunction", "mhc_qkv_norm_rope_fn"]


def _heads(t):
    if t is None:
        return _lib.Heads()
    sb, ss, sh, _ = t.stride()
    return _lib.Heads(t.data_ptr(), sb, ss, sh)


def _check_heads(t, name, like=None, heads=None):
    """A [B, S, heads, d] CUDA tensor of a supported type; returned with unit stride along d."""
    if not torch.is_tensor(t) or t.dim() != 4:
        raise ValueError(f"{name} must be a tensor of shape [B, S, heads, d]")
    if not t.is_cuda:
        raise RuntimeError(f"mhc_ops_b200 runs on CUDA only: {name} is on the CPU (there is no CPU fallback)")
    if t.dtype not in _lib.DTYPES:
        raise TypeError(f"{name} must be bfloat16, float16 or float32, got {t.dtype}")
    if like is not None:
        B, S, _, d = like.shape
        if t.shape[0] != B or t.shape[1] != S or t.shape[3] != d or (heads is not None and t.shape[2] != heads):
            raise ValueError(f"{name} must be [{B}, {S}, {'heads' if heads is None else heads}, {d}], "
                             f"got {tuple(t.shape)}")
        if t.dtype != like.dtype or t.device != like.device:
            raise ValueError(f"{name} is {t.dtype} on {t.device}, expected {like.dtype} on {like.device}")
    return t if t.stride(3) == 1 else t.contiguous()


def _forward_args(q, k, positions, inv_freq, q_weight, k_weight, v, row_scale, eps, interleaved):
    """The checked inputs of either direction: (argument struct, tensors to keep alive, q, k, v)."""
    q = _check_heads(q, "q")
    k = _check_heads(k, "k", like=q)
    if v is not None:
        v = _check_heads(v, "v", like=q)
    B, S, Hq, d = q.shape
    dev = q.device
    inv_freq = _as_f32(inv_freq, dev, "inv_freq")
    rot = 2 * inv_freq.numel()
    if inv_freq.dim() != 1 or rot > d:
        raise ValueError(f"inv_freq must be [rot / 2] with rot <= d = {d}, got {tuple(inv_freq.shape)}")
    if d > 1024:
        raise ValueError(f"d must be at most 1024, got {d}")
    if q_weight is not None:
        q_weight = _as_f32(q_weight, dev, "q_weight")
    if k_weight is not None:
        k_weight = _as_f32(k_weight, dev, "k_weight")
    for w, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if w is not None and w.shape != (d,):
            raise ValueError(f"{name} must be [{d}], got {tuple(w.shape)}")
    if row_scale is not None:
        row_scale = _as_f32(row_scale, dev, "row_scale")
        if row_scale.shape != (B, S):
            raise ValueError(f"row_scale must be [{B}, {S}], got {tuple(row_scale.shape)}")
    psb = pss = pbytes = 0
    if positions is not None:
        if not torch.is_tensor(positions) or positions.dtype not in (torch.int32, torch.int64):
            raise TypeError("positions must be an int32 or int64 tensor")
        if positions.device != dev:
            raise ValueError(f"positions is on {positions.device}, q is on {dev}")
        if positions.shape == (B, S):
            psb, pss = positions.stride()
        elif positions.shape == (S,):
            pss = positions.stride(0)
        else:
            raise ValueError(f"positions must be [{B}, {S}] or [{S}], got {tuple(positions.shape)}")
        pbytes = positions.element_size()
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    args = _lib.QkArgs(
        q=_heads(q), k=_heads(k), v=_heads(v), q_weight=_lib.ptr(q_weight), k_weight=_lib.ptr(k_weight),
        positions=_lib.ptr(positions), inv_freq=_lib.ptr(inv_freq), row_scale=_lib.ptr(row_scale),
        position_batch_stride=psb, position_seq_stride=pss, batch=B, seq=S, q_heads=Hq, k_heads=k.shape[2],
        v_heads=0 if v is None else v.shape[2], d=d, rot=rot, position_bytes=pbytes,
        interleaved=1 if interleaved else 0, dtype=_lib.DTYPES[q.dtype], eps=float(eps))
    return args, (inv_freq, q_weight, k_weight, row_scale, positions), q, k, v


def mhc_qk_norm_rope(q, k, positions, inv_freq, q_weight=None, k_weight=None, *, v=None, row_scale=None,
                     eps: float = 1e-6, interleaved: bool = False):
    """RMSNorm of every query and key head row, then its rotary rotation, in one pass.

    ``q [B,S,Hq,d]``, ``k [B,S,Hk,d]`` and the optional ``v [B,S,Hv,d]`` may be
    views of one packed projection.  ``positions`` are int32/int64 ``[B,S]`` or
    ``[S]`` (None: 0 .. S-1), of any value below 2^31 in magnitude;
    ``inv_freq [rot/2]`` the angles per position of the ``rot <= d`` leading
    elements that turn, in pairs ``(i, i + rot/2)`` or, ``interleaved``,
    ``(2i, 2i + 1)``.  ``q_weight`` / ``k_weight [d]`` are the norms' weights
    (None: ones), ``row_scale [B,S]`` the factor every head of a token is
    multiplied with first.  Returns contiguous ``(q_out, k_out)``, with ``v``
    also ``v_out = row_scale * v``.
    """
    args, keep, q, k, v = _forward_args(q, k, positions, inv_freq, q_weight, k_weight, v, row_scale, eps, interleaved)
    dev = q.device
    outs = [torch.empty(t.shape, dtype=t.dtype, device=dev) for t in (q, k) + (() if v is None else (v,))]
    args.q_out, args.k_out = _heads(outs[0]), _heads(outs[1])
    if v is not None:
        args.v_out = _heads(outs[2])
    with torch.cuda.device(dev):
        _lib.check(_lib.load().mhc_qk_norm_rope(args, torch.cuda.current_stream(dev).cuda_stream), "mhc_qk_norm_rope")
    return tuple(outs)


def _span(t):
    """First byte and the byte behind the last one a strided tensor reaches."""
    lo = t.data_ptr()
    return lo, lo + (sum((n - 1) * st for n, st in zip(t.shape, t.stride())) + 1) * t.element_size()


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
    overlap the inputs or each other.
    """
    fwd, keep, q, k, v = _forward_args(q, k, positions, inv_freq, q_weight, k_weight, v, row_scale, eps, interleaved)
    if (v is None) != (dv_out is None):
        raise ValueError("v and dv_out go together")
    dev, d = q.device, q.shape[3]
    inputs = [q, k] if v is None else [q, k, v]
    names = ("q", "k", "v")
    ups = [_check_heads(g, f"d{n}_out", like=x, heads=x.shape[2])
           for g, x, n in zip((dq_out, dk_out, dv_out), inputs, names)]
    if grad_out is None:
        grads = [torch.empty(x.shape, dtype=x.dtype, device=dev) for x in inputs]
    else:
        grads = list(grad_out)
        if len(grads) != len(inputs):
            raise ValueError(f"grad_out must hold {len(inputs)} tensors")
        for g, x, n in zip(grads, inputs, names):
            _check_heads(g, f"grad_out d{n}", like=x, heads=x.shape[2])
            if g.stride(3) != 1 and d > 1:
                raise ValueError(f"grad_out d{n} must have unit stride along d")
            if any(st == 0 and size > 1 for st, size in zip(g.stride(), g.shape)):
                raise ValueError(f"grad_out d{n} must not be an expanded tensor")
        if q.numel():
            reads = [_span(t) for t in inputs + ups]
            for g, n in zip(grads, names):
                lo, hi = _span(g)
                if any(lo < b and a < hi for a, b in reads):
                    raise ValueError(f"grad_out d{n} overlaps an input")
    f32 = dict(dtype=torch.float32, device=dev)
    dwq = torch.empty(d, **f32) if q_weight is not None and weight_grads else None
    dwk = torch.empty(d, **f32) if k_weight is not None and weight_grads else None
    dsc = torch.empty(q.shape[:2], **f32) if row_scale is not None and row_scale_grad else None
    args = _lib.QkBwdArgs(fwd=fwd, dq_out=_heads(ups[0]), dk_out=_heads(ups[1]), dq=_heads(grads[0]),
                          dk=_heads(grads[1]), dq_weight=_lib.ptr(dwq), dk_weight=_lib.ptr(dwk),
                          d_row_scale=_lib.ptr(dsc))
    if v is not None:
        args.dv_out, args.dv = _heads(ups[2]), _heads(grads[2])
    with torch.cuda.device(dev):
        lib = _lib.load()
        ws = None
        if dwq is not None or dwk is not None:
            nbytes = ctypes.c_size_t(0)
            _lib.check(lib.mhc_qk_norm_rope_bwd_workspace_size(q.shape[0] * q.shape[1], d, ctypes.byref(nbytes)),
                       "mhc_qk_norm_rope_bwd_workspace_size")
            ws = _lib.scratch(nbytes.value, dev)
            args.workspace, args.workspace_bytes = ws.data_ptr(), nbytes.value
        _lib.check(lib.mhc_qk_norm_rope_bwd(args, torch.cuda.current_stream(dev).cuda_stream), "mhc_qk_norm_rope_bwd")
    dv = grads[2] if v is not None else None
    return grads[0], grads[1], dv, dwq, dwk, dsc


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


def mhc_qk_norm_rope_fn(q, k, positions, inv_freq, q_weight=None, k_weight=None, *, v=None, row_scale=None,
                        eps: float = 1e-6, interleaved: bool = False):
    """Differentiable ``mhc_qk_norm_rope``."""
    return MHCQKNormRopeFunction.apply(q, k, positions, inv_freq, q_weight, k_weight, v, row_scale, eps, interleaved)


def mhc_qkv_norm_rope_fn(qkv, q_heads: int, k_heads: int, positions, inv_freq, q_weight=None, k_weight=None, *,
                         row_scale=None, eps: float = 1e-6, interleaved: bool = False):
    """Differentiable ``mhc_qk_norm_rope`` on a packed projection ``[B,S,Hq+2Hk,d]``: returns ``(q, k, v)``."""
    return MHCQKVNormRopeFunction.apply(qkv, q_heads, k_heads, positions, inv_freq, q_weight, k_weight, row_scale,
                                        eps, interleaved)
