"""The float64 statements of oracle/train_oracle.py against autograd and central differences (CPU)."""
import pytest
import torch

from oracle import train_oracle as O


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rot", [(16, 16), (10, 4), (7, 0)])
def test_backward_formula_matches_autograd_and_differences(d, rot, interleaved):
    g = torch.Generator().manual_seed(d)
    B, S, H = 2, 3, 2
    rnd = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)   # noqa: E731
    x, dy, w, sc = rnd(B, S, H, d), rnd(B, S, H, d), 1 + 0.1 * rnd(d), torch.exp(0.2 * rnd(B, S))
    angle = O.angles(torch.tensor([5, 6, 900001]), torch.rand(rot // 2, generator=g), B, S)
    eps = 1e-2   # large enough for the row factor's gradient to show
    leaves = [t.clone().requires_grad_() for t in (x, w, sc)]
    y = O.norm_rope(leaves[0], leaves[1], leaves[2], angle, eps, interleaved)
    auto = torch.autograd.grad(y, leaves, dy)
    mine = O.norm_rope_backward(x, dy, w, sc, angle, eps, interleaved)
    for a, b in zip(auto, mine):
        assert (a - b).abs().max() <= 1e-12 * (1 + b.abs().max())
    # the closed form of the row factor's gradient the kernels use
    z = x * sc[:, :, None, None]
    r = ((z * z).mean(-1, keepdim=True) + eps) ** -0.5
    dn = O.rotate(dy, -angle, interleaved) * w
    closed = eps * (r ** 3 * (dn * x).sum(-1, keepdim=True)).sum((2, 3))
    assert (closed - mine[2]).abs().max() <= 1e-11
    # central differences in a random direction of each input: error ~ h^2
    h = 1e-5
    for i, base in enumerate((x, w, sc)):
        v = rnd(*base.shape)
        args = [x, w, sc]
        f = []
        for sign in (1, -1):
            args[i] = base + sign * h * v
            f.append((O.norm_rope(*args, angle, eps, interleaved) * dy).sum())
        assert abs((f[0] - f[1]) / (2 * h) - (mine[i] * v).sum()) <= 1e-6


def test_newton_schulz_moves_the_singular_values_alone():
    g = torch.Generator().manual_seed(3)
    u = torch.randn(6, 40, generator=g, dtype=torch.float64)
    co = ((3.4445, -4.7750, 2.0315),) * 5
    for t in (u, u.T.contiguous()):
        o = O.newton_schulz(t, co, 1e-7)
        U, s, Vh = torch.linalg.svd(t, full_matrices=False)
        s = s / (t.norm() + 1e-7)
        for a, b, c in co:
            s = a * s + b * s ** 3 + c * s ** 5
        assert (o - (U * s) @ Vh).abs().max() <= 1e-10
        assert 0.6 < s.min() and s.max() < 1.3
