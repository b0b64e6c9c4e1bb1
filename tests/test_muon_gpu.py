"""Newton-Schulz orthogonalisation and the momentum update around it, against float64.

Tolerances.  u32 = 2^-24.  The Gram product and the iteration run in 64 bits, so
O = Q U is left with the rounding of Q to fp32 (1 u32), R products in two chains
(R/2 + 1) and, in the fused update, two more:
  |O - O64| <= (R/2 + 4) u32 sum_k |Q_ik| |U_kj| + u(t) |O|,
plus what 64 bits lose: the Gram sums are off by at most C 2^-53 of the norm
squared, which a step sequence of gain G = prod a_k moves a singular value near
1/G by G^2/2 times (its eigenvalue is 1/G^2 of the norm squared), below
  G^2 C 2^-53 of sum_k |Q_ik| |U_kj|  (G = 485, C = 16384: 4e-7).
"""
import pytest
import torch

from mhc_ops_b200 import NEWTON_SCHULZ_COEFFS, mhc_muon_step, mhc_orthogonalize
from oracle import train_oracle as O

pytestmark = pytest.mark.gpu
U32 = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def _gain(coeffs):
    g = 1.0
    for a, _, _ in coeffs:
        g *= abs(a)
    return g


def _bound(u, want, coeffs, eps=1e-7):
    """sum_k |Q_ik||U_kj| and the tolerance of the module docstring without the output's rounding."""
    tall = u.shape[-2] > u.shape[-1]
    w = (u.mT if tall else u).double()
    lam, V = torch.linalg.eigh(w @ w.mT)
    norm = torch.sqrt((w * w).sum((-2, -1), keepdim=True)) + eps
    s, gain = lam.clamp_min(0).sqrt() / norm[..., 0], torch.ones_like(lam) / norm[..., 0]
    for a, b, c in coeffs:
        f = a + b * s ** 2 + c * s ** 4
        s, gain = s * f, gain * f
    Q = (V * gain[..., None, :]) @ V.mT
    mag = Q.abs() @ w.abs()
    R, C = w.shape[-2:]
    t = ((R / 2 + 4) * U32 + _gain(coeffs) ** 2 * C * 2.0 ** -53) * mag
    return (t.mT if tall else t) + 1e-37


def _gradients(L, R, C, seed, fall=-2.0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    m = min(R, C)
    mix = torch.randn(L, R, m, generator=g, device="cuda") * torch.logspace(0, fall, m, device="cuda")
    return (mix @ torch.randn(L, m, C, generator=g, device="cuda") * 1e-3).to(dtype)


def _near(name, got, want, bound):
    bad = ~((got.double() - want).abs() <= bound)
    assert not bad.any(), (f"{name}: {int(bad.sum())} of {bad.numel()} off, worst "
                           f"{float(((got.double() - want).abs() / bound)[bad].max()):.3g} times the bound")


# (count, rows, cols): the rows of phi for n = 1 .. 8 and what lies between, one column, columns inside a
# chunk, odd widths, more rows than columns, several launches' worth of partial sums
SHAPES = [(1, 3, 16), (1, 8, 1024), (2, 15, 100), (1, 24, 16384), (3, 24, 131), (1, 35, 10005), (2, 48, 640),
          (1, 63, 448), (2, 80, 2048), (1, 80, 81), (1, 1, 1), (1, 1, 5000), (1, 5, 1), (2, 80, 7), (1, 4096, 24),
          (1, 300, 80), (20, 80, 130), (26, 63, 200), (30, 48, 96), (1, 17, 17), (1, 40, 4096), (1, 64, 4100), (1, 9, 33000)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("L,R,C", SHAPES)
def test_orthogonalize_against_float64(L, R, C, dtype):
    u = _gradients(L, R, C, seed=R + C, dtype=dtype)
    got = mhc_orthogonalize(u)
    torch.cuda.synchronize()
    assert got.shape == u.shape and got.dtype == dtype
    want = O.newton_schulz(u, NEWTON_SCHULZ_COEFFS, 1e-7)
    _near("O", got, want, _bound(u, want, NEWTON_SCHULZ_COEFFS) + HALF[dtype] * want.abs())


@pytest.mark.parametrize("coeffs", [((1.5, -0.5, 0.0),), ((3.4445, -4.7750, 2.0315),) * 8 + ((2.0, -1.5, 0.5),) * 2,
                                    ((1.875, -1.25, 0.375),) * 16])
def test_other_coefficients(coeffs):
    u = _gradients(2, 24, 512, seed=4, fall=-1.0)
    got = mhc_orthogonalize(u, coeffs=coeffs, eps=1e-3)
    torch.cuda.synchronize()
    want = O.newton_schulz(u, coeffs, 1e-3)
    tall = _bound(u, want, coeffs, 1e-3)
    _near("O", got, want, tall + U32 * want.abs())


def test_small_singular_values_survive():
    """Singular values down to 1e-5 of the largest: what 32-bit sums of squares would lose."""
    u = _gradients(1, 24, 4096, seed=5, fall=-5.0)
    got = mhc_orthogonalize(u)
    torch.cuda.synchronize()
    want = O.newton_schulz(u, NEWTON_SCHULZ_COEFFS, 1e-7)
    _near("O", got, want, _bound(u, want, NEWTON_SCHULZ_COEFFS) + U32 * want.abs())


def test_zeros_rank_one_huge_tiny_and_nan():
    z = torch.zeros(1, 24, 512, device="cuda")
    one = torch.zeros(1, 24, 512, device="cuda")
    one[0, 3] = torch.randn(512, device="cuda")
    base = _gradients(1, 24, 512, seed=6)
    nan = base.clone()
    nan[0, 0, 0] = float("nan")
    stack = torch.cat([z, one, base * 1e30, base * 1e-12, nan, base])
    got = mhc_orthogonalize(stack)
    torch.cuda.synchronize()
    assert (got[0] == 0).all() and got[4].isnan().all()
    for i in (1, 2, 3, 5):
        want = O.newton_schulz(stack[i], NEWTON_SCHULZ_COEFFS, 1e-7)
        _near(f"matrix {i}", got[i], want, _bound(stack[i], want, NEWTON_SCHULZ_COEFFS) + U32 * want.abs())
    # each matrix alone: the same bits
    for i in (1, 2, 3, 5):
        assert torch.equal(mhc_orthogonalize(stack[i]), got[i])


def test_kinds_of_argument_and_many_matrices():
    u = _gradients(131, 8, 96, seed=7)   # more than one launch takes
    stack = mhc_orthogonalize(u)
    as_list = mhc_orthogonalize(list(u.unbind(0)))
    loose = mhc_orthogonalize([t.clone() for t in u.unbind(0)])
    torch.cuda.synchronize()
    assert isinstance(as_list, list) and len(as_list) == 131
    assert torch.equal(torch.stack(as_list), stack) and torch.equal(torch.stack(loose), stack)
    one = mhc_orthogonalize(u[5])
    strided = mhc_orthogonalize(u[5].T.contiguous().T)   # not contiguous: copied
    torch.cuda.synchronize()
    assert one.shape == (8, 96) and torch.equal(one, strided)
    assert mhc_orthogonalize(torch.empty(0, 8, 96, device="cuda")).shape == (0, 8, 96)
    assert mhc_orthogonalize(torch.empty(8, 0, device="cuda")).shape == (8, 0)


def _muon_inputs(L, R, C, seed, pdt, gdt):
    g = torch.Generator(device="cuda").manual_seed(seed + 100)
    p = (torch.randn(L, R, C, generator=g, device="cuda") / C ** 0.5).to(pdt)
    return p, _gradients(L, R, C, seed, dtype=gdt), _gradients(L, R, C, seed + 1, dtype=torch.float32)


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("pdt,gdt", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                     (torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("L,R,C", [(2, 24, 2048), (1, 35, 1001), (2, 80, 640), (1, 8, 8), (1, 96, 24), (3, 63, 70)])
def test_muon_step_against_float64(L, R, C, pdt, gdt, nesterov):
    p, g, m = _muon_inputs(L, R, C, 11, pdt, gdt)
    lr, mu, wd, scale = 0.3, 0.9, 0.05, 0.7
    p0, m0 = p.clone(), m.clone()
    mhc_muon_step(p, g, m, lr, momentum=mu, nesterov=nesterov, weight_decay=wd, scale=scale)
    torch.cuda.synchronize()
    f32 = lambda v: float(torch.tensor(v, dtype=torch.float32))   # noqa: E731  the coefficients as the kernels hold them
    m64 = mu * m0.double() + (1 - mu) * g.double()
    mag = mu * m0.double().abs() + (1 - mu) * g.double().abs()
    _near("momentum", m, m64, 3 * U32 * mag)   # mu or 1 - mu, a product and the fused sum, a rounding each
    # the direction from the momentum as stored; with nesterov u carries three more roundings, which the iteration
    # (slope at most 1.1 G for these coefficients, twice for the norm) turns into an error spread over the matrix
    u = mu * m.double() + (1 - mu) * g.double() if nesterov else m.double()
    want_o = O.newton_schulz(u, NEWTON_SCHULZ_COEFFS, 1e-7)
    bound = _bound(u, want_o, NEWTON_SCHULZ_COEFFS)
    if nesterov:
        umag = (mu * m.double().abs() + (1 - mu) * g.double().abs())
        spread = 2.2 * _gain(NEWTON_SCHULZ_COEFFS) * 3 * U32 * umag.norm(dim=(-2, -1)) / u.norm(dim=(-2, -1))
        bound = bound + spread[:, None, None]
    keep, step = 1 - f32(lr) * f32(wd), f32(lr) * f32(scale)
    want = keep * p0.double() - step * want_o
    bound = step * (bound + 3 * U32 * want_o.abs()) + 4 * U32 * p0.double().abs() + HALF[pdt] * want.abs()
    _near("param", p, want, bound)


def test_lists_lr_tensor_decay_alone_and_unlisted_neighbours():
    p, g, m = _muon_inputs(4, 24, 256, 21, torch.float32, torch.float32)
    a = [t.clone() for t in (p, g, m)]
    mhc_muon_step(a[0], a[1], a[2], 0.1, weight_decay=0.2)
    lr = torch.full((1,), 0.1, device="cuda")
    ps, ms = list(p.unbind(0)), list(m.unbind(0))
    untouched = p[3].clone(), m[3].clone()
    mhc_muon_step(ps[:3], list(g.unbind(0))[:3], ms[:3], lr, weight_decay=0.2)
    torch.cuda.synchronize()
    assert torch.equal(p[:3], a[0][:3]) and torch.equal(m[:3], a[2][:3])
    assert torch.equal(p[3], untouched[0]) and torch.equal(m[3], untouched[1])
    # no gradient and no momentum: decay alone
    q, z = torch.randn(24, 256, device="cuda"), torch.zeros(24, 256, device="cuda")
    q0 = q.clone()
    mhc_muon_step(q, z, z.clone(), 0.5, weight_decay=0.1)
    torch.cuda.synchronize()
    assert ((q - q0 * 0.95).abs() <= 3 * U32 * q0.abs()).all()


# one launch, a CTA a matrix, a cluster a matrix (ten CTAs, and five when there are many matrices)
@pytest.mark.parametrize("L,R,C", [(3, 24, 512), (3, 24, 2048), (2, 80, 1024), (20, 80, 260)])
def test_determinism_and_captured_schedule(L, R, C):
    p, g, m = _muon_inputs(L, R, C, 31, torch.float32, torch.float32)
    sp, sm, lr = p.clone(), m.clone(), torch.full((1,), 0.1, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        mhc_muon_step(sp, g, sm, lr, weight_decay=0.1)
    ep, em = p.clone(), m.clone()
    for v in (0.1, 0.05, 0.2):
        lr.fill_(v)
        graph.replay()
        mhc_muon_step(ep, g, em, v, weight_decay=0.1)
    torch.cuda.synchronize()
    assert torch.equal(sp, ep) and torch.equal(sm, em)
    del graph


def test_autograd_sees_the_write():
    p = torch.nn.Parameter(torch.randn(8, 32, device="cuda"))
    y = (p * p).sum()
    mhc_muon_step(p, torch.randn(8, 32, device="cuda"), torch.zeros(8, 32, device="cuda"), 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_refusals():
    p, g, m = _muon_inputs(2, 24, 64, 41, torch.float32, torch.float32)
    with pytest.raises(ValueError, match="80 rows"):
        mhc_orthogonalize(torch.zeros(81, 81, device="cuda"))
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        mhc_orthogonalize(torch.zeros(8, 81, device="cuda", dtype=torch.float16))
    with pytest.raises(ValueError, match="coeffs"):
        mhc_orthogonalize(g, coeffs=())
    with pytest.raises(ValueError, match="coeffs"):
        mhc_orthogonalize(g, coeffs=((1.0, 2.0),))
    with pytest.raises(ValueError, match="eps"):
        mhc_orthogonalize(g, eps=0.0)
    with pytest.raises(ValueError, match="eps"):
        mhc_orthogonalize(g, eps=float("nan"))
    with pytest.raises(ValueError, match="must not be an empty"):
        mhc_orthogonalize([])
    with pytest.raises(ValueError, match=r"g\[1\]"):
        mhc_orthogonalize([g[0], g[1][:, :32].contiguous()])
    with pytest.raises(ValueError, match="contiguous"):
        mhc_muon_step(p.mT, g.mT, m.mT, 0.1)
    with pytest.raises(ValueError, match="differ"):
        mhc_muon_step(p, g[:1], m, 0.1)
    with pytest.raises(TypeError, match="momenta must be float32"):
        mhc_muon_step(p, g, m.bfloat16(), 0.1)
    with pytest.raises(ValueError, match="lr must be"):
        mhc_muon_step(p, g, m, torch.zeros(2, device="cuda"))
    for bad in ([p[0], p[0]], [p[0], p.view(-1)[32:32 + 24 * 64].view(24, 64)]):
        with pytest.raises(RuntimeError, match="overlap"):
            mhc_muon_step(bad, list(g.unbind(0)), list(m.unbind(0)), 0.1)
    with pytest.raises(RuntimeError, match="overlap"):
        mhc_muon_step(p, g, g, 0.1)
    before = p.clone()
    mhc_muon_step(list(p.unbind(0)), [g[0], g[0]], list(m.unbind(0)), 0.1)   # gradients are only read
    torch.cuda.synchronize()
    assert not torch.equal(p, before)
