"""Operands, 64-bit plain forms and error bounds for the products with a fused epilogue.

Bounds: the FP32 product is off by at most sqrt(K) * 2^-24 of its terms' magnitudes (the products'
own tolerance); bias and alpha add 4 roundings.  Activations have slopes of at most 1.13 and are
off by a few FP32 units, growing with the exponent's argument: __expf(t) is off by 2 + 1.18 |t|
units, so 16 + 8 |t| units cover it with the divisions.  What is stored as BF16 is off by half a
step more.
"""
from __future__ import annotations

import math

import numpy as np
import torch

import blackhole_b200 as bh
from oracle import oracle as O

U = 2.0 ** -24
FMTS = ("nvfp4", "mxfp4", "mxf8f4")
CALLS = {f: getattr(bh, f + "_bf16_gemm_fused") for f in FMTS}
C0 = math.sqrt(2 / math.pi)


def act64(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "gelu":
        return 0.5 * z * torch.special.erfc(-z / math.sqrt(2))
    if act == "gelu_tanh":
        return z * torch.sigmoid(2 * C0 * (z + 0.044715 * z ** 3))
    if act == "silu":
        return z * torch.sigmoid(z)
    return z


def slope64(z, act):
    if act == "relu":
        return (z > 0).double()
    if act == "gelu":
        return 0.5 * torch.special.erfc(-z / math.sqrt(2)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        t = 2 * C0 * (z + 0.044715 * z ** 3)
        s, r = torch.sigmoid(t), torch.sigmoid(-t)
        return s + z * s * r * 2 * C0 * (1 + 3 * 0.044715 * z * z)
    if act == "silu":
        return torch.sigmoid(z) * (1 + z * torch.sigmoid(-z))
    return torch.ones_like(z)


def act_units(z, act):
    """FP32 units (relative) of an activation's own arithmetic."""
    if act in ("none", "relu"):
        return torch.ones_like(z)
    t = z if act == "silu" else z * z / 2 if act == "gelu" else 2 * C0 * (z + 0.044715 * z ** 3)
    return 16 + 8 * t.abs().clamp(max=200)


_cache = {}


def operands(fmt, M, N, K, seed=0):
    """Quantised operands (host), their 64-bit product and the magnitudes of its terms."""
    key = (fmt, M, N, K, seed)
    if key in _cache:
        return _cache[key]
    xa = O.gen_normal(seed, M * K).reshape(M, K)
    xb = O.gen_normal(seed + 1, N * K, 0.0, 1.5 / math.sqrt(K)).reshape(N, K)
    ka, kb = {"nvfp4": ("nvfp4", "nvfp4"), "mxfp4": ("mxfp4", "mxfp4"), "mxf8f4": ("mxfp8", "mxfp4")}[fmt]
    q = {"nvfp4": O.quantize, "mxfp4": O.quantize_mxfp4, "mxfp8": O.quantize_mxfp8}
    ra, rb = q[ka](xa), q[kb](xb)
    alpha = float(np.float32(ra[2]) * np.float32(rb[2])) if fmt == "nvfp4" else 1.0
    full = []
    for (p, sf), rows, kind in (((ra[0], ra[1]), M, ka), ((rb[0], rb[1]), N, kb)):
        v, s = O.decode_operand(p, sf, rows, K, kind)
        full.append(torch.from_numpy(v).double() * torch.from_numpy(np.repeat(s, K // s.shape[1], 1)).double())
    a, b = full
    r = {"A": ra[0], "SFA": ra[1], "B": rb[0], "SFB": rb[1], "alpha": alpha,
         "prod": alpha * (a @ b.T), "mag": alpha * (a.abs() @ b.abs().T)}
    _cache.clear()
    _cache[key] = r
    return r


def make(fmt, M, N, K, act="none", gated=False, bias=None, residual=False, z=False, beta=1.0, seed=0):
    """A case: operands on the GPU, epilogue inputs and outputs filled with NaN."""
    r = operands(fmt, M, N, K, seed)
    g = torch.Generator().manual_seed(seed + 5)
    n_out = N // 2 if gated else N
    c = dict(fmt=fmt, M=M, N=N, K=K, act=act, gated=gated, beta=beta, alpha=r["alpha"], ref=r)
    for k in ("A", "SFA", "B", "SFB"):
        c[k] = torch.from_numpy(np.ascontiguousarray(r[k])).cuda()
    T = {None: None, "bf16": torch.bfloat16, "f32": torch.float32}[bias]
    c["bias"] = None if T is None else torch.randn(N, generator=g).to(T).cuda()
    c["residual"] = torch.randn(M, n_out, generator=g).to(torch.bfloat16).cuda() if residual else None
    nan = lambda *s: torch.full(s, float("nan"), dtype=torch.bfloat16, device="cuda")  # noqa: E731
    c["D"], c["Z"] = nan(M, n_out), nan(M, N) if z else None
    return c


def call(c, **kw):
    over = dict(D=c["D"])
    over.update({k: kw.pop(k) for k in ("D",) if k in kw})
    args = dict(bias=c["bias"], activation=c["act"], gated=c["gated"], residual=c["residual"], beta=c["beta"],
                Z=c["Z"])
    args.update(kw)
    CALLS[c["fmt"]](c["M"], c["N"], c["K"], c["A"], c["SFA"], c["B"], c["SFB"], over["D"], c["alpha"], **args)


def expected(c):
    """(z, bound of z, D, bound of D) in 64 bits, half a BF16 step not included."""
    r = c["ref"]
    bias = torch.zeros(c["N"], dtype=torch.float64) if c["bias"] is None else c["bias"].cpu().double()
    z = r["prod"] + bias
    ez = U * ((math.sqrt(c["K"]) + 4) * r["mag"] + 4 * (bias.abs() + z.abs()))
    if c["gated"]:
        zg, zu, eg, eu = z[:, 0::2], z[:, 1::2], ez[:, 0::2], ez[:, 1::2]
        a = act64(zg, c["act"])
        u = a * zu
        e = (1.13 * eg + U * act_units(zg, c["act"]) * a.abs()) * (zu.abs() + eu) + a.abs() * eu + U * u.abs()
    else:
        u = act64(z, c["act"])
        e = 1.13 * ez + U * act_units(z, c["act"]) * u.abs()
    if c["residual"] is not None:
        add = c["beta"] * c["residual"].cpu().double()
        u = u + add
        e = e + U * (2 * add.abs() + u.abs())
    return z, ez, u, e


def within(got, ref, err, what=""):
    """|got - ref| <= err + half a step of got's type, everywhere."""
    half = torch.finfo(got.dtype).eps / 2
    got = got.cpu().double()
    assert torch.isfinite(got).all(), what
    tol = err + half * (ref.abs() + err) + 1e-37
    worst = ((got - ref).abs() / tol).max().item()
    assert worst <= 1.0, f"{what}: {worst:.3g} times the bound"


def check(c):
    torch.cuda.synchronize()
    assert bh.device_status(0) == 0
    z, ez, u, e = expected(c)
    within(c["D"], u, e, "D")
    if c["Z"] is not None:
        within(c["Z"], z, ez, "Z")
