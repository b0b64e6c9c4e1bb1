"""The operators around a training step at lengths and widths where a lane keeps sums over many tokens and a matrix
has many columns, against float64."""
import pytest
import torch

from mhc_ops_b200 import (NEWTON_SCHULZ_COEFFS, mhc_muon_step, mhc_orthogonalize, mhc_qk_norm_rope,
                          mhc_qk_norm_rope_backward)
from oracle import train_oracle as O
from tests.test_qkrope_gpu import HALF, TINY, U32, _inputs, _near, _pairs

pytestmark = pytest.mark.gpu


def _check_sums(t, rot, eps, interleaved):
    """All outputs; tolerances of tests/test_qkrope_gpu.py but for the weight gradients' sums.  A lane adds the heads
    of one warp's tokens, at least 148 CTAs of 8 warps sharing them (H T / 1184 terms), then up to 64 lanes and
    warps of a CTA and the CTAs' rows (at most 592 over 8 warps, and 8) are added: H T / 1184 + 150 roundings."""
    q, k, v, sc = t["q"], t["k"], t["v"], t["scale"]
    B, S, _, d = q.shape
    dt, H = q.dtype, q.shape[2] + k.shape[2] + v.shape[2]
    kw = dict(v=v, row_scale=sc, eps=eps, interleaved=interleaved)
    out = mhc_qk_norm_rope(q, k, t["positions"], t["inv_freq"], t["wq"], t["wk"], **kw)
    grads = mhc_qk_norm_rope_backward(q, k, t["positions"], t["inv_freq"], t["dq"], t["dk"], t["wq"], t["wk"],
                                      dv_out=t["dv"], **kw)
    torch.cuda.synchronize()
    angle, s4 = O.angles(t["positions"], t["inv_freq"], B, S), sc.double()[:, :, None, None]
    ds, ds_mag = 0, 0
    for i, (x, dy, w, name) in enumerate(((q, t["dq"], t["wq"], "q"), (k, t["dk"], t["wk"], "k"))):
        x, dy, w = x.double(), dy.double(), w.double()
        y = O.norm_rope(x, w, sc.double(), angle, eps, interleaved)
        a = O.norm_rope(x, w, sc.double(), angle[..., :0], eps, interleaved)
        _near(f"{name}_out", out[i], y, (d / 64 + 24) * U32 * _pairs(a.abs(), rot, interleaved) + HALF[dt] * y.abs()
              + TINY[dt])
        dx, dw, dsx = O.norm_rope_backward(x, dy, w, sc.double(), angle, eps, interleaved)
        r = 1.0 / torch.sqrt(((x * s4) ** 2).mean(-1, keepdim=True) + eps)
        n, dyp = (x * s4 * r).abs(), _pairs(dy.abs(), rot, interleaved)
        m = (w.abs() * dyp * n).mean(-1, keepdim=True)
        _near(f"d{name}", grads[i], dx, (d / 32 + 40) * U32 * s4 * r * (w.abs() * dyp + n * m) + HALF[dt] * dx.abs()
              + TINY[dt])
        _near(f"d{name}_weight", grads[3 + i], dw, (d / 64 + 24 + H * B * S / 1184 + 150) * U32
              * (n * dyp).sum((0, 1, 2)) + 1e-37)
        ds = ds + dsx
        ds_mag = ds_mag + eps * (r ** 3 * (w.abs() * dyp * x.abs()).sum(-1, keepdim=True)).sum((2, 3))
    for name, got, want in (("v_out", out[2], v.double() * s4), ("dv", grads[2], t["dv"].double() * s4)):
        _near(name, got, want, (HALF[dt] + U32) * want.abs() + TINY[dt])
    vdv = v.double() * t["dv"].double()
    _near("drow_scale", grads[5], ds + vdv.sum((2, 3)), (d / 32 + H + 60) * U32 * (ds_mag + vdv.abs().sum((2, 3)))
          + 1e-10)


# whole vectors, half-split and interleaved, one and two rows of lanes; widths and rotations off them
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,S,Hq,Hk,d,rot,interleaved", [(2, 3001, 8, 2, 128, 128, False), (1, 5003, 4, 1, 256, 64, True),
                                                         (3, 2111, 7, 1, 64, 64, False), (2, 2503, 5, 1, 72, 36, False),
                                                         (1, 4999, 3, 1, 50, 50, True)])
def test_long_rope_calls_against_float64(B, S, Hq, Hk, d, rot, interleaved, dtype):
    _check_sums(_inputs(B, S, Hq, Hk, Hk, d, rot, dtype, seed=S), rot, 1e-3, interleaved)


@pytest.mark.parametrize("seed", range(4))
def test_weight_gradients_of_many_rows_keep_their_last_bit(seed):
    """Some 4,700 rows a sum: lanes add a few of them in 32 bits, everything behind the lanes is added in 64.

    What is left are the rounding of a lane's terms and sums, of a CTA's row and of the result, at most u32 of each
    layer's terms and of independent signs: sqrt(3) u32 of the gradient's norm, and with the terms' own errors, which
    average out over the rows, below 2 u32."""
    B, S, d, eps = 2, 333, 64, 1e-6
    t = _inputs(B, S, 7, 1, 1, d, d, torch.float32, seed=100 + seed)
    g = mhc_qk_norm_rope_backward(t["q"], t["k"], t["positions"], t["inv_freq"], t["dq"], t["dk"], t["wq"], t["wk"],
                                  eps=eps)
    torch.cuda.synchronize()
    angle = O.angles(t["positions"], t["inv_freq"], B, S)
    for x, dy, w, got in ((t["q"], t["dq"], t["wq"], g[3]), (t["k"], t["dk"], t["wk"], g[4])):
        want = O.norm_rope_backward(x.double(), dy.double(), w.double(), None, angle, eps, False)[1]
        assert (got - want).norm() <= 2 * U32 * want.norm(), float((got - want).norm() / want.norm() / U32)


def _decided_bound(u, want, coeffs, eps=1e-7):
    """What 64-bit sums and one rounding of the result leave, far below a 32-bit Q or application.

    tests/test_muon_gpu.py has the lift of what the Gram sums lose, G^2 of the norm squared per sum |Q||U|.  An
    accumulator of them takes at most a quarter of the columns (four warps share a chunk at the least), a hundred
    more additions join the accumulators, and the iteration's products add R terms each, three a step, the first of
    which are lifted most: (C / 4 + 100 + 4 R) 2^-53 G^2."""
    from tests.test_muon_gpu import _bound, _gain
    R, C = sorted(u.shape[-2:])
    wide = _bound(u, want, coeffs, eps)   # ((R / 2 + 4) u32 + G^2 C 2^-53) sum |Q||U|
    scale = wide / ((R / 2 + 4) * U32 + _gain(coeffs) ** 2 * C * 2.0 ** -53)
    return (C / 4 + 100 + 4 * R) * 2.0 ** -53 * _gain(coeffs) ** 2 * scale


@pytest.mark.parametrize("L,R,C", [(1, 8, 1024), (2, 24, 512), (1, 24, 4096), (1, 35, 1001), (30, 48, 96), (1, 48, 640),
                                   (2, 63, 500), (2, 80, 640), (20, 80, 130)])
def test_orthogonalised_matrix_is_the_rounded_one(L, R, C):
    from tests.test_muon_gpu import _gradients
    u = _gradients(L, R, C, seed=R * C)
    got = mhc_orthogonalize(u)
    torch.cuda.synchronize()
    want = O.newton_schulz(u, NEWTON_SCHULZ_COEFFS, 1e-7)
    _near("O", got, want, _decided_bound(u, want, NEWTON_SCHULZ_COEFFS) + U32 * want.abs())


def test_update_of_the_wide_configuration_at_its_full_width():
    """n = 8, D = 4096: 80 x 32768, two of them (clusters of ten CTAs) and sixteen (of five)."""
    from tests.test_muon_gpu import _gradients
    R, C, lr, mu, wd = 80, 32768, 0.02, 0.95, 0.1
    for L in (2, 16):
        p, g, m = (_gradients(L, R, C, seed=L + i) for i in range(3))
        p0, m0 = p.clone(), m.clone()
        mhc_muon_step(p, g, m, lr, momentum=mu, nesterov=False, weight_decay=wd)
        torch.cuda.synchronize()
        for i in sorted({0, 1, L - 1}):
            m64 = mu * m0[i].double() + (1 - mu) * g[i].double()
            _near("momentum", m[i], m64, 3 * U32 * (mu * m0[i].double().abs() + (1 - mu) * g[i].double().abs()))
            want_o = O.newton_schulz(m[i], NEWTON_SCHULZ_COEFFS, 1e-7)
            lr32, wd32 = (float(torch.tensor(v, dtype=torch.float32)) for v in (lr, wd))
            keep = 1 - lr32 * wd32
            want = keep * p0[i].double() - lr32 * want_o
            # O rounded to 32 bits and multiplied, the decay's factor twice rounded, the sum
            bound = lr32 * (_decided_bound(m[i], want_o, NEWTON_SCHULZ_COEFFS) + 3 * U32 * want_o.abs())
            _near("param", p[i], want, bound + 4 * U32 * p0[i].double().abs() + U32 * want.abs())


def test_row_factor_carries_a_large_part_of_the_gradient_to_h_in():
    """h_in's gradient is dqkv w - drow_scale rstd^3 h_in / D, against float64 autograd.

    The upstream gradients are the outputs themselves, so that much of dqkv w lies along h_in and the factor's part
    takes it away: as large as what is left.  dqkv and drow_scale are right to some 100 u32 of their terms, the sums of
    512 products in a projection to 512 u32 of theirs at worst, and the terms' sums exceed the sums' norms at most
    30-fold: 1e-3 of the gradient's norm bounds all of it."""
    B, S, D, HQ, HK, d, eps = 2, 48, 256, 4, 2, 64, 0.3
    g = torch.Generator(device="cuda").manual_seed(7)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")   # noqa: E731
    f = (10000.0 ** (-torch.arange(d // 2, device="cuda") / (d // 2))).float()
    h, w = rnd(B, S, D), rnd((HQ + 2 * HK) * d, D) / D ** 0.5
    rstd, parts = 1.0 / torch.sqrt((h * h).mean(-1) + 1e-6), (HQ, HK, HK)
    q, k, v = (h @ w.T).view(B, S, -1, d).split(parts, dim=2)
    up = mhc_qk_norm_rope(q, k, None, f, v=v, row_scale=rstd, eps=eps)
    dqkv = torch.empty(B, S, sum(parts), d, device="cuda")
    out = mhc_qk_norm_rope_backward(q, k, None, f, up[0], up[1], v=v, dv_out=up[2], row_scale=rstd, eps=eps,
                                    grad_out=dqkv.split(parts, dim=2))
    direct = dqkv.flatten(2).double() @ w.double()
    through = -(out[5][..., None] * rstd[..., None] ** 3 * h / D).double()
    x = h.double().requires_grad_()
    y = ((x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6)) @ w.double().T).view(B, S, -1, d)
    angle = O.angles(None, f, B, S)
    o = [O.norm_rope(t, None, None, angle, eps, False) for t in y.split(parts, dim=2)[:2]] + [y[:, :, HQ + HK:]]
    want, = torch.autograd.grad(o, x, [t.double() for t in up])
    assert through.norm() >= 0.5 * want.norm(), float(through.norm() / want.norm())
    assert (direct + through - want).norm() <= 1e-3 * want.norm()
    assert (direct - want).norm() >= 0.49 * want.norm()
