"""Cases of the training-step operators around the hyper-connection pre-op, for timing and comparison.

Four operators:

* ``rope_fwd`` -- per-head RMSNorm of queries and keys with the rotary position rotation in the same pass, the
  row factor of the RMSNorm before the projection (``h_in_rstd`` of ``mhc_forward_pre_fused_norm``) and the values
  scaled by it;
* ``rope_bwd`` -- its gradients: one packed gradient of the projection's output, the norm weights' and the row
  factor's;
* ``ortho`` -- Newton-Schulz orthogonalisation of a list of gradients of phi;
* ``muon`` -- the whole update of a list of phi: momentum, orthogonalisation, weight decay, in place.

``own`` selects between the plain form (elementary torch operations in 32 bits, 64 where those lose what matters)
and the library's calls.
"""
from __future__ import annotations

import math

import torch

own = False

# The usual five quintic steps of the orthogonalisation.
COEFFS = ((3.4445, -4.7750, 2.0315),) * 5
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------ cases
def _rope(name, op, B, S, Hq, Hk, d, rot, dtype="bf16", interleaved=False, scaled=False, weights=True, far=4096,
          base=10000.0):
    return {"name": name, "op": op, "B": B, "S": S, "Hq": Hq, "Hk": Hk, "d": d, "rot": rot, "dtype": dtype,
            "interleaved": interleaved, "scaled": scaled, "weights": weights, "far": far, "base": base}


def _mat(name, op, L, R, C, dtype="fp32", nesterov=True):
    return {"name": name, "op": op, "L": L, "R": R, "C": C, "dtype": dtype, "nesterov": nesterov}


def listed():
    return [
        # one sequence decoding one token: launch latency
        _rope("rope_fwd_one_token", "rope_fwd", 1, 1, 32, 8, 128, 128, far=32768),
        # a serving batch, one new token each, at far positions; norm before the projection folded in
        _rope("rope_fwd_batch_step", "rope_fwd", 512, 1, 32, 8, 128, 128, scaled=True, far=1 << 20, base=500000.0),
        # ragged prefill, partial rotation, a head width that is no power of two
        _rope("rope_fwd_ragged", "rope_fwd", 3, 1237, 12, 4, 96, 48, dtype="fp16", interleaved=True),
        # the bench's training batch (B=4, S=4096, D=4096 = 32 heads of 128)
        _rope("rope_fwd_train", "rope_fwd", 4, 4096, 32, 8, 128, 128, scaled=True),
        # a small fp32 batch, one shared key head
        _rope("rope_bwd_small_fp32", "rope_bwd", 2, 333, 7, 1, 64, 64, dtype="fp32", interleaved=True, scaled=True),
        # wide heads, a long single sequence, no row factor
        _rope("rope_bwd_wide_heads", "rope_bwd", 1, 8191, 16, 2, 256, 64, far=1 << 17),
        # the bench's training batch, backward
        _rope("rope_bwd_train", "rope_bwd", 4, 4096, 32, 8, 128, 128, scaled=True),
        # phi of a small two-stream model: launch latency
        _mat("ortho_n2_D512", "ortho", 1, 8, 1024),
        # one phi of the bench's model (n=4, D=4096)
        _mat("ortho_n4_D4096", "ortho", 1, 24, 16384),
        # bf16 gradients of a few five-stream layers, odd width
        _mat("ortho_n5_ragged_bf16", "ortho", 6, 35, 10005, dtype="bf16"),
        # every phi of 32 layers with two sublayers each (n=4, D=4096)
        _mat("muon_n4_64_layers", "muon", 64, 24, 16384),
        # the wide configuration (n=8, D=4096), eight of them
        _mat("muon_n8_8_layers", "muon", 8, 80, 32768),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope_fwd", "rope_bwd", "ortho", "muon"])
    if op.startswith("rope"):
        d = rng.choice([32, 50, 64, 72, 80, 96, 112, 128, 128, 192, 256])
        rot = rng.choice([d, d, d // 2, d // 4]) // 2 * 2
        Hk = rng.choice([1, 2, 3, 4, 8])
        Hq = Hk * rng.choice([1, 2, 4, 5, 8])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        size = 4 if dtype == "fp32" else 2
        limit = 4 * 4096 * 48 * 128 * 2 // ((Hq + 2 * Hk) * d * size)
        tokens = min(_log(rng, 1, 16384), limit)
        B = min(tokens, _log(rng, 1, 64))
        S = max(1, tokens // B)
        return _rope("", op, B, S, Hq, Hk, d, rot, dtype, rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.8,
                     _log(rng, max(2, S), 1 << 20), rng.choice([10000.0, 500000.0]))
    n = rng.randint(1, 8)
    R = n * n + 2 * n
    C = n * _log(rng, 8, 4096)
    room = min(20_000_000 // (R * C), 8 * 80 * 80 * 32768 // (R * R * C))
    L = min(_log(rng, 1, 64), max(1, room))
    return _mat("", op, L, R, C, rng.choice(["fp32", "fp32", "bf16"]), rng.random() < 0.7)


# ------------------------------------------------------------------------------------------------ inputs
def _randn(shape, g, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _rope_inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, S, Hq, Hk, d = c["B"], c["S"], c["Hq"], c["Hk"], c["d"]
    dt = DTYPES[c["dtype"]]
    st = {"case": c}
    # a projection's output: heads of differing size
    heads = Hq + 2 * Hk
    st["qkv"] = (torch.randn((B, S, heads, d), generator=g, device="cuda")
                 * torch.exp(0.5 * torch.randn((heads, 1), generator=g, device="cuda"))).to(dt)
    # each sequence goes on from where it stands
    start = torch.randint(0, max(1, c["far"] - S + 1), (B, 1), generator=g, device="cuda")
    st["positions"] = start + torch.arange(S, device="cuda")
    half = c["rot"] // 2
    st["inv_freq"] = (c["base"] ** (-torch.arange(half, device="cuda", dtype=torch.float64) / max(1, half))).float()
    if c["weights"]:
        st["wq"] = 1.0 + _randn((d,), g, scale=0.1)
        st["wk"] = 1.0 + _randn((d,), g, scale=0.1)
    else:
        st["wq"] = st["wk"] = None
    st["scale"] = torch.exp(0.3 * torch.randn((B, S), generator=g, device="cuda")) if c["scaled"] else None
    if c["op"] == "rope_bwd":
        st["dq"] = _randn((B, S, Hq, d), g, dt)
        st["dk"] = _randn((B, S, Hk, d), g, dt)
        st["dv"] = _randn((B, S, Hk, d), g, dt)
    return st


def _mat_inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    L, R, C = c["L"], c["R"], c["C"]
    dt = DTYPES[c["dtype"]]
    st = {"case": c}

    def gradient(scale):
        # a few strong directions and a tail, as the gradient of a small matrix over many tokens has
        m = min(R, C)
        fall = torch.logspace(0, -2, m, device="cuda")
        mix = torch.randn((L, R, m), generator=g, device="cuda") * fall
        return torch.matmul(mix, torch.randn((L, m, C), generator=g, device="cuda")) * (scale / math.sqrt(m))

    st["grad"] = list(gradient(1e-3).to(dt).unbind(0))
    if c["op"] == "muon":
        # the layers' matrices, kept in one allocation each
        st["momenta"] = gradient(5e-4)
        st["params"] = (torch.randn((L, R, C), generator=g, device="cuda") / math.sqrt(C)).to(dt)
        st["momentum"], st["param"] = list(st["momenta"].unbind(0)), list(st["params"].unbind(0))
    return st


def prepare(case, seed):
    return _rope_inputs(case, seed) if case["op"].startswith("rope") else _mat_inputs(case, seed)


# ------------------------------------------------------------------------------------------------ plain forms
def _split(qkv, c):
    return qkv[:, :, :c["Hq"]], qkv[:, :, c["Hq"]:c["Hq"] + c["Hk"]], qkv[:, :, c["Hq"] + c["Hk"]:]


def _cos_sin(st):
    a = st["positions"].double()[..., None] * st["inv_freq"].double()   # far positions need 64 bits
    return a.cos().float()[:, :, None], a.sin().float()[:, :, None]


def _rotate(x, cos, sin, interleaved):
    rot = 2 * cos.shape[-1]
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack((a * cos - b * sin, a * sin + b * cos), dim=-1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat((a * cos - b * sin, a * sin + b * cos), dim=-1)
    return torch.cat((y, x[..., rot:]), dim=-1)


EPS = 1e-6


def _plain_rope_fwd(st):
    c = st["case"]
    cos, sin = _cos_sin(st)
    q, k, v = _split(st["qkv"], c)
    out = []
    for x, w in ((q, st["wq"]), (k, st["wk"])):
        z = x.float()
        if st["scale"] is not None:
            z = z * st["scale"][:, :, None, None]
        z = z * torch.rsqrt((z * z).mean(-1, keepdim=True) + EPS)
        if w is not None:
            z = z * w
        out.append(_rotate(z, cos, sin, c["interleaved"]).to(x.dtype))
    if st["scale"] is not None:
        out.append((v.float() * st["scale"][:, :, None, None]).to(v.dtype))
    return out


def _plain_rope_bwd(st):
    c = st["case"]
    cos, sin = _cos_sin(st)
    q, k, v = _split(st["qkv"], c)
    s = st["scale"]
    s4 = None if s is None else s[:, :, None, None]
    grads, dws, ds = [], [], None
    for x, dy, w in ((q, st["dq"], st["wq"]), (k, st["dk"], st["wk"])):
        x = x.float()
        z = x if s is None else x * s4
        r = torch.rsqrt((z * z).mean(-1, keepdim=True) + EPS)
        n = z * r
        da = _rotate(dy.float(), cos, -sin, c["interleaved"])
        if w is None:
            dn = da
        else:
            dws.append((da * n).sum((0, 1, 2)))
            dn = da * w
        dz = r * (dn - n * (dn * n).mean(-1, keepdim=True))
        grads.append(dz if s is None else dz * s4)
        if s is not None:
            part = EPS * (r ** 3 * (dn * x).sum(-1, keepdim=True)).sum((2, 3))
            ds = part if ds is None else ds + part
    dv = st["dv"].float()
    if s is not None:
        ds = ds + (v.float() * dv).sum((2, 3))
        dv = dv * s4
        grads.append(dv)
    dqkv = torch.cat(grads, dim=2).to(st["qkv"].dtype)
    return [dqkv] + dws + ([] if s is None else [ds])


def _plain_newton_schulz(u):
    # in 64 bits: five steps raise what 32 bits lose of a gradient's small singular values a few hundred times
    tall = u.shape[-2] > u.shape[-1]
    x = (u.mT if tall else u).double()
    x = x / ((x * x).sum((-2, -1), keepdim=True).sqrt() + 1e-7)
    for a, b, cc in COEFFS:
        A = torch.matmul(x, x.mT)
        x = a * x + torch.matmul(b * A + cc * torch.matmul(A, A), x)
    return (x.mT if tall else x).float()


MU, LR, DECAY = 0.95, 0.02, 0.1


def _plain_muon(st):
    g = torch.stack([t.float() for t in st["grad"]])
    params, momenta = st["params"], st["momenta"]
    momenta.copy_(MU * momenta + (1 - MU) * g)
    u = MU * momenta + (1 - MU) * g if st["case"]["nesterov"] else momenta
    params.copy_(params.float() * (1 - LR * DECAY) - LR * _plain_newton_schulz(u))
    return [params, momenta]


def run(state):
    op = state["case"]["op"]
    if own:
        return _run_own(state, op)
    if op == "rope_fwd":
        return _plain_rope_fwd(state)
    if op == "rope_bwd":
        return _plain_rope_bwd(state)
    if op == "ortho":
        u = torch.stack([t.float() for t in state["grad"]])
        return list(_plain_newton_schulz(u).to(state["grad"][0].dtype).unbind(0))
    return _plain_muon(state)


# ------------------------------------------------------------------------------------------------ the library's calls
def _run_own(st, op):
    import mhc_ops_b200 as M
    c = st["case"]
    if op == "rope_fwd":
        q, k, v = _split(st["qkv"], c)
        return list(M.mhc_qk_norm_rope(q, k, st["positions"], st["inv_freq"], st["wq"], st["wk"],
                                       v=v if c["scaled"] else None, row_scale=st["scale"], eps=EPS,
                                       interleaved=c["interleaved"]))
    if op == "rope_bwd":
        q, k, v = _split(st["qkv"], c)
        heads = c["Hq"] + (2 if c["scaled"] else 1) * c["Hk"]
        dqkv = torch.empty((c["B"], c["S"], heads, c["d"]), dtype=st["qkv"].dtype, device="cuda")
        dq, dk, dv = _split(dqkv, c)
        scaled = c["scaled"]
        out = M.mhc_qk_norm_rope_backward(q, k, st["positions"], st["inv_freq"], st["dq"], st["dk"], st["wq"],
                                          st["wk"], v=v if scaled else None, dv_out=st["dv"] if scaled else None,
                                          row_scale=st["scale"], eps=EPS, interleaved=c["interleaved"],
                                          grad_out=(dq, dk, dv) if scaled else (dq, dk))
        return [dqkv] + [t for t in out[3:] if t is not None]
    if op == "ortho":
        return list(M.mhc_orthogonalize(st["grad"], coeffs=COEFFS, eps=1e-7))
    M.mhc_muon_step(st["param"], st["grad"], st["momentum"], lr=LR, momentum=MU, nesterov=c["nesterov"],
                    weight_decay=DECAY, coeffs=COEFFS, eps=1e-7)
    return [st["params"], st["momenta"]]


# ------------------------------------------------------------------------------------------------ work
def work(case):
    c = case
    if c["op"].startswith("rope"):
        T, d = c["B"] * c["S"], c["d"]
        size = 4 if c["dtype"] == "fp32" else 2
        heads = c["Hq"] + (2 if c["scaled"] else 1) * c["Hk"]
        row = T * heads * d * size
        small = T * (8 + (4 if c["scaled"] else 0)) + 2 * c["rot"] + (8 * d if c["weights"] else 0)
        if c["op"] == "rope_fwd":
            return {"bytes": 2 * row + small, "flops": 9 * T * heads * d}
        return {"bytes": 3 * row + small + (8 * d if c["weights"] else 0) + (4 * T if c["scaled"] else 0),
                "flops": 18 * T * heads * d}
    L, R, C = c["L"], min(c["R"], c["C"]), max(c["R"], c["C"])
    size = 4 if c["dtype"] == "fp32" else 2
    flops = L * (R * (R + 1) * C + 2 * R * R * C)
    if c["op"] == "ortho":
        return {"bytes": 2 * L * R * C * size, "flops": flops}
    # gradient read; momentum and parameter read and written
    return {"bytes": L * R * C * (size + 8 + 2 * size), "flops": flops + 8 * L * R * C}


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_rope_heads(x, s, w, turn, interleaved):
    """One side's outputs in 64 bits: the pairs as complex numbers, turned by exp(i angle)."""
    z = x if s is None else x * s[:, :, None, None]
    z = z / torch.sqrt(torch.mean(torch.square(z), dim=3, keepdim=True) + EPS)
    if w is not None:
        z = z * w.double()
    half = turn.shape[-1]
    head, tail = z[..., :2 * half], z[..., 2 * half:]
    if interleaved:
        p = torch.complex(head[..., 0::2].contiguous(), head[..., 1::2].contiguous()) * turn
        head = torch.view_as_real(p).reshape(head.shape)
    else:
        p = torch.complex(head[..., :half].contiguous(), head[..., half:].contiguous()) * turn
        head = torch.cat((p.real, p.imag), dim=3)
    return torch.cat((head, tail), dim=3)


def _exact_rope(c, seed):
    st = _rope_inputs(c, seed)
    angle = st["positions"].double().unsqueeze(-1) * st["inv_freq"].double()
    turn = torch.polar(torch.ones_like(angle), angle).unsqueeze(2)
    backward = c["op"] == "rope_bwd"
    Hq, Hk = c["Hq"], c["Hk"]
    leaves = []

    def leaf(t):
        t = t.double()
        if backward:
            t.requires_grad_()
            leaves.append(t)
        return t

    used = st["qkv"] if c["scaled"] else st["qkv"][:, :, :Hq + Hk]
    qkv = leaf(used)
    wq = None if st["wq"] is None else leaf(st["wq"])
    wk = None if st["wk"] is None else leaf(st["wk"])
    s = None if st["scale"] is None else leaf(st["scale"])
    out = [_exact_rope_heads(qkv[:, :, :Hq], s, wq, turn, c["interleaved"]),
           _exact_rope_heads(qkv[:, :, Hq:Hq + Hk], s, wk, turn, c["interleaved"])]
    if s is not None:
        out.append(qkv[:, :, Hq + Hk:] * s[:, :, None, None])
    if not backward:
        return out
    ups = [st["dq"].double(), st["dk"].double()] + ([st["dv"].double()] if s is not None else [])
    return list(torch.autograd.grad(out, leaves, ups))


def _exact_newton_schulz(u):
    """The iteration on the eigenvalues of the smaller Gram matrix: a step with factor a + b s^2 + c s^4 multiplies
    each singular value s by it and leaves the singular vectors."""
    tall = u.shape[0] > u.shape[1]
    w = u.t() if tall else u
    lam, V = torch.linalg.eigh(w @ w.t())
    s = lam.clamp_min(0).sqrt() / (u.square().sum().sqrt() + 1e-7)
    gain = torch.ones_like(s) / (u.square().sum().sqrt() + 1e-7)
    for a, b, cc in COEFFS:
        factor = a + s.square() * (b + cc * s.square())
        s, gain = s * factor, gain * factor
    out = (V * gain) @ (V.t() @ w)
    return out.t() if tall else out


def _exact_mat(c, seed):
    st = _mat_inputs(c, seed)
    if c["op"] == "ortho":
        return [_exact_newton_schulz(t.double()) for t in st["grad"]]
    params, moms = [], []
    for p, g, m in zip(st["param"], st["grad"], st["momentum"]):
        g = g.double()
        m = MU * m.double() + (1 - MU) * g
        u = m + (1 - MU) * (g - m) if c["nesterov"] else m
        params.append(p.double() - LR * (DECAY * p.double() + _exact_newton_schulz(u)))
        moms.append(m)
    return [torch.stack(params), torch.stack(moms)]


def exact(case, seed):
    return _exact_rope(case, seed) if case["op"].startswith("rope") else _exact_mat(case, seed)
