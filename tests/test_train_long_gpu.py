"""The operators around a training step at lengths and widths where a lane keeps sums over many tokens and a matrix
has many columns, against float64."""
import pytest
import torch

from mhc_ops_b200 import mhc_qk_norm_rope, mhc_qk_norm_rope_backward
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
