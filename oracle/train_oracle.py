"""float64 statements of the operators around a training step that the reference has no counterpart of:
the per-head norms of queries and keys with the rotary rotation, and the orthogonalised momentum update.
Test infrastructure; torch in float64, written from the formulas alone."""
from __future__ import annotations

from decimal import Decimal, getcontext
from fractions import Fraction

import torch


def rotate(x, angle, interleaved):
    """The first 2 * angle.shape[-1] elements of each row turned pairwise; x [B,S,H,d], angle [B,S,half]."""
    half = angle.shape[-1]
    c, s = torch.cos(angle)[:, :, None], torch.sin(angle)[:, :, None]
    y = x.clone()
    ia = torch.arange(half, device=x.device) * 2 if interleaved else torch.arange(half, device=x.device)
    ib = ia + 1 if interleaved else ia + half
    y[..., ia] = x[..., ia] * c - x[..., ib] * s
    y[..., ib] = x[..., ia] * s + x[..., ib] * c
    return y


def angles(positions, inv_freq, B, S):
    if positions is None:
        positions = torch.arange(S, device=inv_freq.device)
    return positions.double().expand(B, S)[..., None] * inv_freq.double()


def norm_rope(x, w, scale, angle, eps, interleaved):
    """One side's forward; every argument float64 (w, scale may be None)."""
    z = x if scale is None else x * scale[:, :, None, None]
    a = z / torch.sqrt((z * z).mean(-1, keepdim=True) + eps)
    return rotate(a if w is None else a * w, angle, interleaved)


def norm_rope_backward(x, dy, w, scale, angle, eps, interleaved):
    """One side's gradients by the formula: (dx, dw, dscale, and the sums of magnitudes the tolerances need)."""
    s = 1.0 if scale is None else scale[:, :, None, None]
    z = x * s
    r = 1.0 / torch.sqrt((z * z).mean(-1, keepdim=True) + eps)
    n = z * r
    da = rotate(dy, -angle, interleaved)
    dn = da if w is None else da * w
    m = (dn * n).mean(-1, keepdim=True)
    dx = s * r * (dn - n * m)
    dw = (da * n).sum((0, 1, 2))
    ds = (x * r * (dn - n * m)).sum((2, 3))
    return dx, dw, ds


def newton_schulz(u, coeffs, eps):
    """The iteration as it is written, on the matrix itself."""
    tall = u.shape[-2] > u.shape[-1]
    x = (u.mT if tall else u).double()
    x = x / (torch.sqrt((x * x).sum((-2, -1), keepdim=True)) + eps)
    for a, b, c in coeffs:
        A = x @ x.mT
        x = a * x + (b * A + c * (A @ A)) @ x
    return x.mT if tall else x


def muon_step(p, g, m, lr, mu, nesterov, decay, scale, coeffs, eps):
    """(new parameter, new momentum) in float64."""
    g, m, p = g.double(), m.double(), p.double()
    m = mu * m + (1 - mu) * g
    u = mu * m + (1 - mu) * g if nesterov else m
    return (1 - lr * decay) * p - lr * scale * newton_schulz(u, coeffs, eps), m


def _inverse_two_pi():
    """1 / (2 pi) to 60 digits, pi = 16 arctan(1/5) - 4 arctan(1/239)."""
    getcontext().prec = 70

    def arctan(n):
        term = total = Decimal(1) / n
        k = 1
        while abs(term) > Decimal(10) ** -66:
            term, k = -term / (n * n), k + 2
            total += term / k
        return total

    return Fraction(1 / (8 * (4 * arctan(5) - arctan(239))))


def far_angles(positions, inv_freq):
    """position * inv_freq [len(positions), len(inv_freq)], reduced to [-pi, pi] in exact arithmetic: the angles of
    positions at which a float64 product has lost what float32 needs."""
    inv = _inverse_two_pi()
    rows = []
    for f in inv_freq.tolist():
        g = Fraction(f) * inv
        rows.append([float(t - round(t)) for t in (g * int(p) for p in positions.tolist())])
    return torch.tensor(rows, dtype=torch.float64).T * (2 * torch.pi)
