"""Per-head norms of queries and keys with the rotary rotation, against float64.

Tolerances.  u32 = 2^-24 is half a step of fp32, u(t) that of the output type.
Forward: a sum of squares of d terms (at most 16 per lane and 5 shuffles, or
d/32 and 5) loses at most (d/32 + 21) u32, half of it reaches the row's factor;
scaling, weighting, the factor's own rounding and the division by d add 6, cos
and sin (2 units in the last place and the angle's rounding) 4, the turn 2:
  |y - y64| <= (d/64 + 24) u32 (|a_i| + |a_j|) + u(t) |y|,  a the pair before the turn.
Backward: da as above without the norm (6 u32 (|dy_i| + |dy_j|)); dx = s r (dn - n m)
with m a mean of d products, (d/32 + 24) u32 mean|dn n| off:
  |dx - dx64| <= (d/32 + 40) u32 s r (|w| (|dy_i| + |dy_j|) + |n| mean(|w| (|dy_i| + |dy_j|) |n|)) + u(t) |dx|.
Weight gradients add at most H rows of a token per lane (one token a warp here:
tokens < 2368), then 5 shuffles, 8 warps and the CTAs' rows (at most 37 and 8):
  (d/64 + 24 + H + 60) u32 sum(|n| (|dy_i| + |dy_j|)).
Row factor: eps r^3 sum(dn x) + sum(v dv): the sums as above, three times r's error:
  (d/32 + H + 60) u32 (eps r^3 sum(|w| (|dy_i| + |dy_j|) |x|) + sum|v dv|).
"""
import pytest
import torch

from mhc_ops_b200 import (mhc_qk_norm_rope, mhc_qk_norm_rope_backward, mhc_qk_norm_rope_fn, mhc_qkv_norm_rope_fn)
from oracle import train_oracle as O

pytestmark = pytest.mark.gpu
U32 = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 1e-38, torch.float16: 2.0 ** -25, torch.float32: 1e-38}   # half the smallest subnormal step


def _inputs(B, S, Hq, Hk, Hv, d, rot, dtype, seed, far=1 << 20, weights=True, scale=True, pos="bs"):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")   # noqa: E731
    t = {"qkv": (rnd(B, S, Hq + Hk + Hv, d) * torch.exp(0.5 * rnd(Hq + Hk + Hv, 1))).to(dtype)}
    t["q"], t["k"], t["v"] = t["qkv"].split((Hq, Hk, Hv), dim=2)
    if Hv == 0:
        t["v"] = None
    t["inv_freq"] = (10000.0 ** (-torch.arange(rot // 2, device="cuda") / max(1, rot // 2))).float()
    start = torch.randint(0, far, (B, 1), generator=g, device="cuda")
    t["positions"] = {"bs": start + torch.arange(S, device="cuda"), "s32": torch.arange(S, device="cuda").int() + 7,
                      "none": None}[pos]
    t["wq"], t["wk"] = (1 + 0.2 * rnd(d), 1 + 0.2 * rnd(d)) if weights else (None, None)
    t["scale"] = torch.exp(0.5 * rnd(B, S)) if scale else None
    t["dq"], t["dk"] = rnd(B, S, Hq, d).to(dtype), rnd(B, S, Hk, d).to(dtype)
    t["dv"] = rnd(B, S, Hv, d).to(dtype) if Hv else None
    return t


def _pairs(mag, rot, interleaved):
    """|a_i| + |a_j| of each element's pair (its own magnitude outside the turned part)."""
    out = mag.clone()
    half = rot // 2
    ia = torch.arange(half, device=mag.device) * (2 if interleaved else 1)
    ib = ia + 1 if interleaved else ia + half
    s = mag[..., ia] + mag[..., ib]
    out[..., ia], out[..., ib] = s, s
    return out


def _d(t):
    return None if t is None else t.double()


def _near(name, got, want, bound):
    bad = ~((got.double() - want).abs() <= bound)
    assert not bad.any(), (f"{name}: {int(bad.sum())} of {bad.numel()} off, worst "
                           f"{float(((got.double() - want).abs() / bound)[bad].max()):.3g} times the bound")


def _check(t, rot, eps=1e-6, interleaved=False, call=None):
    q, k, v, sc = t["q"], t["k"], t["v"], t["scale"]
    B, S, _, d = q.shape
    dt = q.dtype
    kw = dict(v=v, row_scale=sc, eps=eps, interleaved=interleaved)
    out = mhc_qk_norm_rope(q, k, t["positions"], t["inv_freq"], t["wq"], t["wk"], **kw)
    grads = mhc_qk_norm_rope_backward(q, k, t["positions"], t["inv_freq"], t["dq"], t["dk"], t["wq"], t["wk"],
                                      dv_out=t["dv"], **kw)
    torch.cuda.synchronize()
    angle = O.angles(t["positions"], t["inv_freq"], B, S)
    s4 = 1.0 if sc is None else sc.double()[:, :, None, None]
    H = q.shape[2] + k.shape[2] + (0 if v is None else v.shape[2])
    ds = torch.zeros(B, S, dtype=torch.float64, device="cuda")
    ds_mag = torch.zeros_like(ds)
    for i, (x, dy, w, name) in enumerate(((q, t["dq"], t["wq"], "q"), (k, t["dk"], t["wk"], "k"))):
        x, dy, w = x.double(), dy.double(), _d(w)
        y = O.norm_rope(x, w, _d(sc), angle, eps, interleaved)
        a = O.norm_rope(x, w, _d(sc), angle[..., :0], eps, interleaved)
        assert out[i].shape == x.shape and out[i].dtype == dt and out[i].is_contiguous()
        _near(f"{name}_out", out[i], y, (d / 64 + 24) * U32 * _pairs(a.abs(), rot, interleaved) + HALF[dt] * y.abs()
              + TINY[dt])
        dx, dw, dsx = O.norm_rope_backward(x, dy, w, _d(sc), angle, eps, interleaved)
        ww = torch.ones(d, dtype=torch.float64, device="cuda") if w is None else w.abs()
        r = 1.0 / torch.sqrt(((x * s4) ** 2).mean(-1, keepdim=True) + eps)
        n = (x * s4 * r).abs()
        dyp = _pairs(dy.abs(), rot, interleaved)
        m = (ww * dyp * n).mean(-1, keepdim=True)
        _near(f"d{name}", grads[i], dx, (d / 32 + 40) * U32 * s4 * r * (ww * dyp + n * m) + HALF[dt] * dx.abs()
              + TINY[dt])
        if w is None:
            assert grads[3 + i] is None
        else:
            assert grads[3 + i].dtype == torch.float32
            _near(f"d{name}_weight", grads[3 + i], dw, (d / 64 + 84 + H) * U32 * (n * dyp).sum((0, 1, 2)) + 1e-37)
        ds += dsx
        ds_mag += eps * (r ** 3 * (ww * dyp * x.abs()).sum(-1, keepdim=True)).sum((2, 3))
    if v is not None:
        want = v.double() * s4
        _near("v_out", out[2], want, (HALF[dt] + U32) * want.abs() + TINY[dt])
        want = t["dv"].double() * s4
        _near("dv", grads[2], want, (HALF[dt] + U32) * want.abs() + TINY[dt])
        ds += (v.double() * t["dv"].double()).sum((2, 3))
        ds_mag += (v.double() * t["dv"].double()).abs().sum((2, 3))
    if sc is None:
        assert grads[5] is None
    else:
        # the oracle's direct sum of the eps term cancels in float64 too: 2^-50 of its terms
        _near("drow_scale", grads[5], ds, (d / 32 + H + 60) * U32 * ds_mag + 1e-10)


# (B, S, Hq, Hk, Hv, d, rot): every lane layout of the vector kernels, partial rotations, one token,
# one head, heads that do not fill a warp
VEC = [(1, 1, 32, 8, 8, 128, 128), (2, 37, 6, 2, 2, 64, 64), (1, 65, 5, 1, 1, 96, 32), (3, 7, 3, 3, 3, 80, 80),
       (1, 130, 4, 1, 0, 256, 64), (2, 9, 2, 1, 1, 512, 512), (1, 33, 9, 3, 1, 16, 16), (1, 300, 1, 1, 0, 32, 0),
       (5, 3, 16, 16, 16, 192, 96)]
# widths, rotations and sizes that take the other kernels
ANY = [(1, 1, 1, 1, 1, 1, 0), (2, 5, 3, 1, 1, 2, 2), (1, 17, 4, 2, 2, 50, 24), (1, 19, 2, 1, 0, 72, 36),
       (2, 3, 2, 1, 1, 1000, 1000), (1, 4, 1, 1, 1, 1024, 512), (1, 40, 7, 1, 1, 33, 10)]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", VEC + ANY, ids=str)
def test_against_float64(shape, dtype, interleaved):
    _check(_inputs(*shape, dtype, seed=sum(shape)), shape[-1], interleaved=interleaved)


def test_interleaved_rotation_that_ends_inside_a_lane():
    _check(_inputs(2, 11, 3, 1, 1, 64, 22, torch.bfloat16, seed=1), 22, interleaved=True)


@pytest.mark.parametrize("weights,scale,pos", [(False, False, "none"), (True, False, "s32"), (False, True, "bs")])
@pytest.mark.parametrize("d,rot", [(128, 128), (50, 24)])
def test_options(weights, scale, pos, d, rot):
    _check(_inputs(2, 40, 4, 2, 2, d, rot, torch.bfloat16, seed=5, weights=weights, scale=scale, pos=pos), rot)


@pytest.mark.parametrize("eps", [0.0, 1e-2])
def test_eps(eps):
    _check(_inputs(2, 40, 4, 2, 2, 64, 64, torch.float32, seed=6), 64, eps=eps)


@pytest.mark.parametrize("d", [128, 50])
def test_many_tokens(d):
    """More tokens than one round of the grid, so lanes keep sums over several; checked against the same call in parts."""
    t = _inputs(3, 1500, 8, 2, 2, d, d // 2 * 2, torch.bfloat16, seed=8)
    args = lambda i, j: (t["q"][i:j], t["k"][i:j], t["positions"][i:j], t["inv_freq"], t["dq"][i:j], t["dk"][i:j],   # noqa: E731
                         t["wq"], t["wk"])
    kw = lambda i, j: dict(v=t["v"][i:j], dv_out=t["dv"][i:j], row_scale=t["scale"][i:j])   # noqa: E731
    whole = mhc_qk_norm_rope_backward(*args(0, 3), **kw(0, 3))
    parts = [mhc_qk_norm_rope_backward(*args(i, i + 1), **kw(i, i + 1)) for i in range(3)]
    for j in (0, 1, 2):
        assert torch.equal(whole[j], torch.cat([p[j] for p in parts])), j
    # how many warps share a token, and so the order its heads are added in, goes by the number of tokens: two sums
    # of the module docstring's bound each (the eps term is below 1 here: eps r^3 |x| <= eps r^2 sqrt(d) is tiny)
    mag = (t["v"].double() * t["dv"].double()).abs().sum((2, 3)) + 1
    _near("drow_scale", whole[5], torch.cat([p[5] for p in parts]).double(), 2 * (d / 32 + 12 + 60) * U32 * mag)
    for j in (3, 4):
        total = sum(p[j].double() for p in parts)
        # sums of n terms of magnitude about 1 in two orders: rows 4500 x heads; each lane adds
        # 4500 * 10 / (148 * 2 * 8) ~ 20 of them, then 110 more partial sums
        n = t["q"].shape[2] * 4500
        assert ((whole[j].double() - total).abs() <= 2 * 160 * U32 * n).all(), j
    again = mhc_qk_norm_rope_backward(*args(0, 3), **kw(0, 3))
    torch.cuda.synchronize()
    for a, b in zip(whole, again):
        assert torch.equal(a, b)


def test_strides_layouts_and_written_slices():
    """Inputs of another axis order and alignment; gradients written into a packed tensor, its other parts untouched."""
    t = _inputs(2, 21, 4, 2, 2, 64, 64, torch.bfloat16, seed=9)
    ref = mhc_qk_norm_rope_backward(t["q"].contiguous(), t["k"].contiguous(), t["positions"], t["inv_freq"], t["dq"],
                                    t["dk"], t["wq"], t["wk"], row_scale=t["scale"])
    ref_f = mhc_qk_norm_rope(t["q"].contiguous(), t["k"].contiguous(), t["positions"], t["inv_freq"], t["wq"], t["wk"],
                             row_scale=t["scale"])
    by_head = lambda x: x.transpose(1, 2).contiguous().transpose(1, 2)   # noqa: E731  [B,H,S,d] in memory
    pack = torch.full((2, 21, 8, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    got = mhc_qk_norm_rope_backward(by_head(t["q"]), t["k"], t["positions"], t["inv_freq"], by_head(t["dq"]),
                                    by_head(t["dk"]), t["wq"], t["wk"], row_scale=t["scale"],
                                    grad_out=(pack[:, :, :4], pack[:, :, 5:7]))
    got_f = mhc_qk_norm_rope(by_head(t["q"]), t["k"], t["positions"], t["inv_freq"], t["wq"], t["wk"],
                             row_scale=t["scale"])
    torch.cuda.synchronize()
    assert got[0].data_ptr() == pack.data_ptr()
    for i in (0, 1, 3, 4, 5):
        assert torch.equal(got[i], ref[i]), i
    for a, b in zip(got_f, ref_f):
        assert torch.equal(a, b)
    assert (pack[:, :, 4] == 7).all() and (pack[:, :, 7] == 7).all()
    # rows that start 2 bytes off a 16-byte boundary, an element stride of 2, an expanded input: the same values
    # within the float64 bound
    odd = torch.zeros(2 * 21 * 8 * 65 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(2, 21, 8, 65)[..., :64]
    odd.copy_(t["qkv"])
    u = dict(t, q=odd[:, :, :4], k=odd[:, :, 4:6], v=odd[:, :, 6:])
    _check(u, 64)
    wide = torch.zeros(2, 21, 8, 128, dtype=torch.bfloat16, device="cuda")
    wide[..., ::2] = t["qkv"]
    u = dict(t, q=wide[:, :, :4, ::2], k=wide[:, :, 4:6, ::2], v=wide[:, :, 6:, ::2])
    _check(u, 64)
    u = dict(t, k=t["k"][:, :1, :1].expand(2, 21, 2, 64))
    _check(u, 64)


def test_rows_of_zeros_infinities_and_nan_stay_in_their_rows():
    for d in (128, 50):
        t = _inputs(1, 6, 2, 1, 1, d, d // 2 * 2, torch.float32, seed=11)
        clean = mhc_qk_norm_rope(t["q"], t["k"], t["positions"], t["inv_freq"], t["wq"], t["wk"], v=t["v"])
        q = t["q"].clone()
        q[0, 1, 0] = 0.0
        q[0, 2, 1, 3] = float("nan")
        q[0, 3, 0, 5] = float("inf")
        dirty = mhc_qk_norm_rope(q, t["k"], t["positions"], t["inv_freq"], t["wq"], t["wk"], v=t["v"])
        torch.cuda.synchronize()
        assert (dirty[0][0, 1, 0] == 0).all() and dirty[0][0, 2, 1].isnan().all() and dirty[0][0, 3, 0].isnan().any()
        touched = torch.zeros(1, 6, 2, dtype=torch.bool, device="cuda")
        touched[0, 1, 0] = touched[0, 2, 1] = touched[0, 3, 0] = True
        assert torch.equal(dirty[0][~touched], clean[0][~touched])
        assert torch.equal(dirty[1], clean[1]) and torch.equal(dirty[2], clean[2])


def test_far_and_negative_positions():
    t = _inputs(1, 4, 2, 1, 1, 64, 64, torch.float32, seed=12)
    t["positions"] = torch.tensor([[(1 << 31) - 1, -(1 << 31) + 1, 0, -5]], device="cuda")
    # the angle itself: position * inv_freq in 64 bits, 2^-53 of up to 2^31 / 2 pi turns twice, under 2^-24
    _check(t, 64)


def test_no_tokens():
    t = _inputs(2, 0, 2, 1, 1, 64, 64, torch.bfloat16, seed=13)
    out = mhc_qk_norm_rope(t["q"], t["k"], None, t["inv_freq"], t["wq"], t["wk"], v=t["v"])
    g = mhc_qk_norm_rope_backward(t["q"], t["k"], None, t["inv_freq"], t["dq"], t["dk"], t["wq"], t["wk"])
    torch.cuda.synchronize()
    assert [tuple(o.shape) for o in out] == [(2, 0, 2, 64), (2, 0, 1, 64), (2, 0, 1, 64)]
    assert (g[3] == 0).all() and (g[4] == 0).all()


def test_autograd_packed_and_apart():
    t = _inputs(2, 30, 4, 2, 2, 64, 32, torch.bfloat16, seed=14)
    ref = mhc_qk_norm_rope_backward(t["q"], t["k"], t["positions"], t["inv_freq"], t["dq"], t["dk"], t["wq"], t["wk"],
                                    v=t["v"], dv_out=t["dv"], row_scale=t["scale"])
    leaf = lambda x: x.detach().clone().requires_grad_()   # noqa: E731
    qkv, wq, wk, sc = leaf(t["qkv"]), leaf(t["wq"]), leaf(t["wk"]), leaf(t["scale"])
    q, k, v = mhc_qkv_norm_rope_fn(qkv, 4, 2, t["positions"], t["inv_freq"], wq, wk, row_scale=sc)
    torch.autograd.backward([q, k, v], [t["dq"], t["dk"], t["dv"]])
    assert torch.equal(qkv.grad, torch.cat(ref[:3], dim=2))
    for a, b in ((wq, ref[3]), (wk, ref[4]), (sc, ref[5])):
        assert torch.equal(a.grad, b)
    q1, k1, v1 = leaf(t["q"]), leaf(t["k"]), leaf(t["v"])
    wq, sc = leaf(t["wq"]), leaf(t["scale"])
    outs = mhc_qk_norm_rope_fn(q1, k1, t["positions"], t["inv_freq"], wq, t["wk"], v=v1, row_scale=sc)
    torch.autograd.backward(outs, [t["dq"], t["dk"], t["dv"]])
    for a, b in ((q1, ref[0]), (k1, ref[1]), (v1, ref[2]), (wq, ref[3]), (sc, ref[5])):
        assert torch.equal(a.grad, b)
    # one output unused: its upstream gradient is zero
    q2 = leaf(t["q"])
    qo, ko = mhc_qk_norm_rope_fn(q2, t["k"], t["positions"], t["inv_freq"], t["wq"])
    qo.backward(t["dq"])
    torch.cuda.synchronize()
    assert q2.grad.abs().sum() > 0


def test_captured_step_and_a_second_stream():
    t = _inputs(1, 70, 4, 2, 2, 128, 128, torch.bfloat16, seed=15)

    def step(t):
        kw = dict(v=t["v"], row_scale=t["scale"])
        return (mhc_qk_norm_rope(t["q"], t["k"], t["positions"], t["inv_freq"], t["wq"], t["wk"], **kw)
                + mhc_qk_norm_rope_backward(t["q"], t["k"], t["positions"], t["inv_freq"], t["dq"], t["dk"], t["wq"],
                                            t["wk"], dv_out=t["dv"], **kw))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graphs = []
    for _ in range(2):   # two graphs of the same stream, replayed on two streams: no scratch is shared
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs = step(t)
        graphs.append((g, outs))
    fresh = _inputs(1, 70, 4, 2, 2, 128, 128, torch.bfloat16, seed=16)
    for key in ("qkv", "positions", "wq", "wk", "scale", "dq", "dk", "dv"):
        t[key].copy_(fresh[key])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graphs[0][0].replay()
    with torch.cuda.stream(side):
        graphs[1][0].replay()
    torch.cuda.synchronize()
    ref = step(fresh)
    torch.cuda.synchronize()
    for _, outs in graphs:
        for a, b in zip(outs, ref):
            assert torch.equal(a, b)
    del graphs


def test_refusals():
    t = _inputs(1, 4, 2, 1, 1, 64, 64, torch.bfloat16, seed=17)
    f = t["inv_freq"]
    ok = dict(q=t["q"], k=t["k"], positions=t["positions"], inv_freq=f)
    call = lambda **kw: mhc_qk_norm_rope(**{**ok, **kw})   # noqa: E731
    with pytest.raises(ValueError, match="shape"):
        call(q=t["q"][0])
    with pytest.raises(TypeError, match="bfloat16, float16 or float32"):
        call(q=t["q"].double())
    with pytest.raises(ValueError, match="k "):
        call(k=t["k"].float())
    with pytest.raises(ValueError, match="k must be"):
        call(k=t["k"][:, :3])
    with pytest.raises(ValueError, match="inv_freq"):
        call(inv_freq=torch.ones(33, device="cuda"))
    with pytest.raises(ValueError, match="inv_freq is on"):
        call(inv_freq=f.cpu())
    with pytest.raises(TypeError, match="positions"):
        call(positions=t["positions"].float())
    with pytest.raises(ValueError, match="positions must be"):
        call(positions=t["positions"][:, :2])
    with pytest.raises(ValueError, match="q_weight must be"):
        call(q_weight=torch.ones(32, device="cuda"))
    with pytest.raises(ValueError, match="row_scale must be"):
        call(row_scale=torch.ones(4, device="cuda"))
    with pytest.raises(ValueError, match="eps"):
        call(eps=-1.0)
    wide = torch.zeros(1, 1, 1, 1032, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="at most 1024"):
        call(q=wide, k=wide, positions=None)
    back = lambda **kw: mhc_qk_norm_rope_backward(t["q"], t["k"], t["positions"], f, t["dq"], t["dk"], **kw)   # noqa: E731
    with pytest.raises(ValueError, match="go together"):
        back(v=t["v"])
    with pytest.raises(ValueError, match="overlaps"):
        back(grad_out=(t["dq"], torch.empty_like(t["dk"])))
    with pytest.raises(ValueError, match="hold 2"):
        back(grad_out=(t["dq"],))
    with pytest.raises(ValueError, match="expanded"):
        back(grad_out=(torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16, device="cuda").expand(1, 4, 2, 64),
                       torch.empty_like(t["dk"])))


def test_shape_errors_of_the_registered_operators_are_exceptions():
    """Their messages name sizes; torch.ops.mhc.fwd's among them."""
    from mhc_ops_b200 import ops
    x = torch.zeros(1, 4, 2, 16, dtype=torch.bfloat16, device="cuda")
    z = lambda *s: torch.zeros(*s, device="cuda")   # noqa: E731
    with pytest.raises(RuntimeError, match=r"phi must be \[8, 32\], got \[8, 31\]"):
        ops.fwd(x, z(8, 31), z(3), z(8))
