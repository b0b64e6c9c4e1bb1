"""The angles of the rotation at near and far positions, against exact arithmetic.

The first element of every pair is 1 and the second 0, with eps = 1/2, so that a
row's factor is 1 up to its rounding and the outputs are cos and sin.  u32 =
2^-24.  sincospi is right to 2 units in the last place, 4 u32 of its value; the
turn by the angle's rounding adds half a unit, 1 u32, and the row's factor
another 1 (its own error is common to both).  So cos and sin are off by at most
6 u32 of themselves, and the angle they stand for by
  |y_c sin - y_s cos| <= 12 u32 |sin cos| <= 6 u32.
"""
import numpy as np
import pytest
import torch

from mhc_ops_b200 import mhc_qk_norm_rope
from oracle import train_oracle as O

pytestmark = pytest.mark.gpu
U32 = 2.0 ** -24


def _frequencies(half, rng):
    """Frequencies below 1 whose product with 1 / 2 pi a float64 holds worst."""
    f = np.sort(rng.uniform(0.5, 1.0, 4096).astype(np.float32))
    inv = O._inverse_two_pi()
    lost = [abs(float(O.Fraction(float(x)) * inv - O.Fraction(float(x) * float(inv)))) for x in f]
    return torch.from_numpy(f[np.argsort(lost)[-half:]].copy())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d", [128, 50])
@pytest.mark.parametrize("low,high", [(-64, 64), (1 << 20, 1 << 21), ((1 << 31) - (1 << 20), 1 << 31),
                                      (-(1 << 31) + 1, -(1 << 31) + (1 << 20))])
def test_cos_and_sin_against_exact_arithmetic(d, interleaved, low, high):
    rng = np.random.default_rng(3)
    f = _frequencies(d // 2, rng)
    pos = torch.from_numpy(rng.integers(low, high, 512))
    x = torch.zeros(1, 512, 1, d, device="cuda")
    first = slice(0, d, 2) if interleaved else slice(0, d // 2)
    second = slice(1, d, 2) if interleaved else slice(d // 2, d)
    x[..., first] = 1.0
    y, _ = mhc_qk_norm_rope(x, x, pos.cuda(), f.cuda(), eps=0.5, interleaved=interleaved)
    torch.cuda.synchronize()
    y = y[0, :, 0].double().cpu()
    a = O.far_angles(pos, f)
    off = (y[:, first] * a.sin() - y[:, second] * a.cos()).abs() / U32
    assert off.max() <= 6, float(off.max())
    # the row's factor: rsqrt to 2 units in the last place, 4 u32, and half a unit of the sum of squares' d terms
    size = (y[:, first] ** 2 + y[:, second] ** 2 - 1).abs()
    assert size.max() <= 2 * (6 + 4 + d / 64 + 24) * U32
