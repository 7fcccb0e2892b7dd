"""Measured workloads of the operators around the block-scaled products: the products with a
fused epilogue (bias, activation or gated activation, residual), the gradient through that
epilogue, and the norms before and after a block fused with its gate and residual scale,
forward (BF16, FP32 or the next product's quantised operand) and backward.

`run` computes a case in plain FP32 torch operations, or, where `own` is true, by the
framework's calls; `exact` computes it in 64 bits, written apart from the plain form.
"""
import math

import torch

own = False

DEV = "cuda"
BF16 = torch.bfloat16
FORMATS = ("nvfp4", "mxfp4", "mxf8f4")
ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu")


# ---------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------
def _gemm(name, fmt, M, N, K, act, gated=False, bias="none", residual=False, z=False):
    return {"name": name, "op": "gemm", "fmt": fmt, "M": M, "N": N, "K": K, "act": act,
            "gated": gated, "bias": bias, "residual": residual, "z": z}


def _gback(name, M, N, act, gated=False):
    return {"name": name, "op": "gemm_backward", "M": M, "N": N, "act": act, "gated": gated}


def _norm(name, op, rows, H, kind, stream, post, gate_rows, out="bf16"):
    # gate_rows: -1 no gate, 0 one gate row for all, g > 0 one gate row per g rows
    return {"name": name, "op": op, "rows": rows, "H": H, "kind": kind, "stream": stream,
            "post": post, "gate_rows": gate_rows, "out": out}


def listed():
    return [
        # one token through the gate/up projection of a decoder's MLP (the decode shape)
        _gemm("decode_1_gated", "nvfp4", 1, 28672, 8192, "silu", gated=True),
        # a small decode batch through the down projection, MXFP8 activations, residual added
        _gemm("decode_16_down", "mxf8f4", 16, 8192, 28672, "none", residual=True),
        # a ragged batch of short requests: odd M, N off the tile, K with a tail, FP32 bias
        _gemm("ragged_203", "mxfp4", 203, 5000, 4128, "gelu", bias="f32", residual=True),
        # a training step's projection that keeps its pre-activations for the backward pass
        _gemm("train_2048", "mxf8f4", 2048, 8192, 2048, "gelu_tanh", bias="bf16", z=True),
        # a prompt through the down projection with bias and residual (the prefill shape)
        _gemm("prefill_16384_down", "nvfp4", 16384, 8192, 28672, "none", bias="bf16", residual=True),
        # gradient through the epilogue: a small odd layer, and a large gated one
        _gback("epilogue_grad_odd", 333, 1000, "gelu"),
        _gback("epilogue_grad_gated", 8192, 28672, "silu", gated=True),
        # one decoded token between attention and MLP: post norm, gate, residual, pre norm
        _norm("norm_token", "norm", 1, 8192, "rms", "bf16", True, 0),
        # conditioned layer norm over a padded batch of odd sequences, FP32 residual stream
        _norm("norm_layer_f32", "norm", 1239, 5120, "layer", "f32", False, 413),
        # a prompt's residual, gate and norm straight to the next product's MXFP8 operand
        _norm("norm_prompt_mxfp8", "norm", 16384, 8192, "rms", "bf16", True, 0, "mxfp8"),
        # training: odd rows and width, layer norms with a gate per sequence
        _norm("norm_grad_odd", "norm_backward", 345, 1000, "layer", "f32", True, 115),
        # training: a large batch, RMS norms before and after, one learned gate vector
        _norm("norm_grad_large", "norm_backward", 16384, 8192, "rms", "bf16", True, 0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("gemm", "gemm", "gemm_backward", "norm", "norm", "norm_backward"))
    if op == "gemm":
        fmt, gated = rng.choice(FORMATS), rng.random() < 0.4
        kstep, nstep = (128 if fmt == "mxf8f4" else 32), (16 if gated else 8)
        while True:
            M = _log(rng, 1, 16384)
            N = max(1, _log(rng, 256, 28672) // nstep) * nstep
            K = max(1, _log(rng, 256, 28672) // kstep) * kstep
            if M * N * K <= 16384 * 8192 * 28672:
                break
        c = _gemm("", fmt, M, N, K, rng.choice(ACTS), gated, rng.choice(("none", "f32", "bf16")),
                  rng.random() < 0.5, rng.random() < 0.25)
    elif op == "gemm_backward":
        gated = rng.random() < 0.5
        c = _gback("", _log(rng, 1, 8192), max(2, _log(rng, 256, 28672) // 16) * 16,
                   rng.choice(ACTS), gated)
    else:
        out = rng.choice(("bf16", "bf16", "f32", "mxfp8")) if op == "norm" else "bf16"
        step = 32 if out == "mxfp8" else 8
        rows = _log(rng, 1, 16384)
        c = _norm("", op, rows, max(2, _log(rng, 256, 16384 if rows <= 8192 else 8192) // step) * step,
                  rng.choice(("rms", "layer")), rng.choice(("bf16", "f32")), rng.random() < 0.5,
                  rng.choice((-1, 0, 1, max(1, rows // 3))), out)
    del c["name"]
    return c


# ---------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(g, *shape, dtype=torch.float32, std=1.0, mean=0.0):
    return torch.empty(shape, dtype=torch.float32, device=DEV).normal_(mean, std, generator=g).to(dtype)


def _pow2(e):
    """2^e as FP32 for integer e in [-126, 127], built from its bits (exact)."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _e2m1_codes(v):
    """Nearest E2M1 codes (ties to the even code, saturating), packed two per byte."""
    a = v.abs()
    m = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5)
         + (a >= 3.5) + (a > 5.0)).to(torch.uint8)
    m |= (v < 0).to(torch.uint8) << 3
    return m[:, 0::2] | (m[:, 1::2] << 4)


def _blocked(sf):
    """[rows, groups] scale bytes -> the 128x4 blocked layout (rows and groups zero-padded)."""
    r, g = sf.shape
    rp, gp = -(-r // 128) * 128, -(-g // 4) * 4
    out = torch.zeros((rp, gp), dtype=torch.uint8, device=sf.device)
    out[:r, :g] = sf
    return out.view(rp // 128, 4, 32, gp // 4, 4).permute(0, 3, 2, 1, 4).contiguous().view(-1)


def _mx_exponent(y, emax):
    """Shared exponents floor(log2 amax) - emax of the last axis' blocks, from the bits."""
    bits = y.abs().amax(-1).view(torch.int32)
    e = (bits >> 23) - 127 - emax
    return torch.where(bits >> 23 == 0, torch.full_like(e, -127), e).clamp_(-127, 127)


def _quantise(x, fmt):
    """FP32 [rows, K] -> (codes, scale factors in the blocked layout, global scale)."""
    rows, K = x.shape
    if fmt == "nvfp4":
        g = float(x.abs().max()) / 2688.0
        b = x.view(rows, K // 16, 16)
        s = (b.abs().amax(-1) / 6.0 / g).clamp_(max=448.0).to(torch.float8_e4m3fn)
        scale = (s.float() * g).unsqueeze(-1)
        q = torch.where(scale > 0, b / scale, torch.zeros_like(b)).view(rows, K)
        return _e2m1_codes(q), _blocked(s.view(torch.uint8)), g
    b = x.view(rows, K // 32, 32)
    e = _mx_exponent(b, 8 if fmt == "mxfp8" else 2)
    q = (b * _pow2(-e.clamp(-127, 126)).unsqueeze(-1)).view(rows, K)
    sf = _blocked((e + 127).to(torch.uint8))
    if fmt == "mxfp8":
        return q.clamp_(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8), sf, 1.0
    return _e2m1_codes(q), sf, 1.0


def _operand(g, rows, K, fmt, std, outliers):
    """A quantised [rows, K] operand of N(0, std) values, made in pieces of rows."""
    if fmt != "nvfp4":
        piece = max(128, (1 << 26) // K // 128 * 128)
    else:
        piece = rows                       # one global scale for the whole tensor
    parts = []
    for r in range(0, rows, piece):
        x = _randn(g, min(piece, rows - r), K, std=std)
        if outliers:                       # one feature in a hundred is 20 times as large
            x[:, torch.randperm(K, generator=g, device=DEV)[: max(1, K // 100)]] *= 20
        parts.append(_quantise(x, fmt))
        del x
    return torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts]), parts[0][2]


def prepare(case, seed):
    g, c = _gen(seed), case
    s = dict(c)
    if c["op"] == "gemm":
        M, N, K = c["M"], c["N"], c["K"]
        a_fmt = "mxfp8" if c["fmt"] == "mxf8f4" else c["fmt"]
        b_fmt = "mxfp4" if c["fmt"] == "mxf8f4" else c["fmt"]
        s["A"], s["SFA"], ga = _operand(g, M, K, a_fmt, 1.0, True)
        s["B"], s["SFB"], gb = _operand(g, N, K, b_fmt, 0.02, False)
        s["alpha"] = ga * gb
        n_out = N // 2 if c["gated"] else N
        s["bias_t"] = None if c["bias"] == "none" else _randn(
            g, N, std=0.5, dtype=BF16 if c["bias"] == "bf16" else torch.float32)
        s["res"] = _randn(g, M, n_out, dtype=BF16) if c["residual"] else None
        s["D"] = torch.empty((M, n_out), dtype=BF16, device=DEV)
        s["Z"] = torch.empty((M, N), dtype=BF16, device=DEV) if c["z"] else None
    elif c["op"] == "gemm_backward":
        M, N = c["M"], c["N"]
        s["Z"] = _randn(g, M, N, dtype=BF16, std=1.5)
        s["dD"] = _randn(g, M, N // 2 if c["gated"] else N, dtype=BF16, std=1e-2)
        s["dZ"] = torch.empty((M, N), dtype=BF16, device=DEV)
        s["dbias"] = torch.empty(N, device=DEV)
    else:
        rows, H, T = c["rows"], c["H"], BF16 if c["stream"] == "bf16" else torch.float32
        x = _randn(g, rows, H)
        x[:, torch.randperm(H, generator=g, device=DEV)[: max(1, H // 200)]] *= 10
        s["x"] = x.to(T)
        del x
        s["o"] = _randn(g, rows, H, dtype=BF16, std=0.5)
        if c["kind"] == "layer":
            s["o"] += 0.1
        for k in ("w", "wp"):
            s[k] = _randn(g, H, std=0.1, mean=1.0)
        for k in ("b", "bp"):
            s[k] = _randn(g, H, std=0.1) if c["kind"] == "layer" else None
        if not c["post"]:
            s["wp"] = s["bp"] = None
        s["scale"] = 0.7
        gr = c["gate_rows"]
        s["gate"] = None if gr < 0 else _randn(g, -(-rows // gr) if gr else 1, H, dtype=BF16)
        if c["op"] == "norm":
            s["h"] = torch.empty_like(s["x"])
            if c["out"] == "mxfp8":
                s["y"] = torch.empty((rows, H), dtype=torch.uint8, device=DEV)
                s["sf"] = torch.empty(-(-rows // 128) * -(-H // 128) * 512, dtype=torch.uint8, device=DEV)
            else:
                s["y"] = torch.empty((rows, H), device=DEV, dtype=BF16 if c["out"] == "bf16" else torch.float32)
                s["sf"] = None
        else:
            # what the forward pass left behind: the new stream and the rows' statistics
            h, stats, _ = _norm_parts(s)
            s["h"], s["stats"] = h.to(T), stats
            s["dy"] = _randn(g, rows, H, dtype=BF16, std=1e-2)
            s["dh"] = _randn(g, rows, H, dtype=T, std=1e-2)
            s["dx"] = torch.empty_like(s["dh"])
            s["do"] = torch.empty((rows, H), dtype=BF16, device=DEV)
            f = lambda on: torch.empty(H, device=DEV) if on else None  # noqa: E731
            layer = c["kind"] == "layer"
            s["dw"], s["db"] = f(True), f(layer)
            s["dwp"], s["dbp"] = f(c["post"]), f(c["post"] and layer)
            s["dgate"] = None if gr < 0 else torch.empty(s["gate"].shape, device=DEV)
    return s


# ---------------------------------------------------------------------------------------
# Plain form, FP32
# ---------------------------------------------------------------------------------------
def _unblocked(sf, rows, groups):
    rp, gp = -(-rows // 128) * 128, -(-groups // 4) * 4
    return sf.view(rp // 128, gp // 4, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(rp, gp)[:rows, :groups]


_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _values(q, sf, rows, K, fmt):
    """The FP32 values that a quantised operand stands for (the global scale apart)."""
    vec = 16 if fmt == "nvfp4" else 32
    scales = _unblocked(sf, rows, K // vec)
    scales = scales.view(torch.float8_e4m3fn).float() if fmt == "nvfp4" else scales.view(torch.float8_e8m0fnu).float()
    if fmt == "mxfp8":
        v = q.view(torch.float8_e4m3fn).float()
    else:
        lut = torch.tensor(_E2M1, device=q.device)
        v = torch.stack((lut[(q & 15).int()], lut[(q >> 4).int()]), -1)
    return (v.view(rows, K // vec, vec) * scales.unsqueeze(-1)).view(rows, K)


_C = math.sqrt(2.0 / math.pi)


def _act(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "gelu":
        return 0.5 * z * torch.erfc(z * -math.sqrt(0.5))
    if act == "gelu_tanh":
        return z / (1 + torch.exp(-2 * _C * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * torch.erfc(z * -math.sqrt(0.5)) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        s = 1 / (1 + torch.exp(-2 * _C * (z + 0.044715 * z * z * z)))
        return s + z * s * (1 - s) * 2 * _C * (1 + 3 * 0.044715 * z * z)
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


def _plain_gemm(s):
    a_fmt = "mxfp8" if s["fmt"] == "mxf8f4" else s["fmt"]
    b_fmt = "mxfp4" if s["fmt"] == "mxf8f4" else s["fmt"]
    a = _values(s["A"], s["SFA"], s["M"], s["K"], a_fmt)
    b = _values(s["B"], s["SFB"], s["N"], s["K"], b_fmt)
    z = s["alpha"] * (a @ b.T)
    del a, b
    if s["bias_t"] is not None:
        z = z + s["bias_t"].float()
    u = _act(z[:, 0::2], s["act"]) * z[:, 1::2] if s["gated"] else _act(z, s["act"])
    if s["res"] is not None:
        u = u + s["res"].float()
    out = {"D": u.to(BF16)}
    if s["z"]:
        out["Z"] = z.to(BF16)
    return out


def _plain_gemm_backward(s):
    z, d = s["Z"].float(), s["dD"].float()
    if s["gated"]:
        gate, up = z[:, 0::2], z[:, 1::2]
        g = torch.stack((d * up * _act_slope(gate, s["act"]), d * _act(gate, s["act"])), -1).view(z.shape)
    else:
        g = d * _act_slope(z, s["act"])
    return {"dZ": g.to(BF16), "dbias": g.sum(0, dtype=torch.float64).float()}


def _stats(v, kind):
    mu = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[:, :1])
    return mu, ((v - mu).square().mean(-1, keepdim=True) + 1e-6).rsqrt()


def _gate_of(s, rows):
    """The gate row of each row, FP32."""
    gr = s["gate_rows"]
    g = s["gate"].float()
    if gr == 0:
        return g
    return g if gr == 1 else g.repeat_interleave(gr, 0)[:rows]


def _norm_parts(s):
    """The new stream, the rows' statistics [rows, 4] and the normed result, FP32."""
    x, p = s["x"].float(), s["o"].float()
    mp = rp = torch.zeros_like(x[:, :1])
    if s["post"]:
        mp, rp = _stats(p, s["kind"])
        p = (p - mp) * rp * s["wp"]
        if s["bp"] is not None:
            p = p + s["bp"]
    if s["gate"] is not None:
        p = p * _gate_of(s, x.shape[0])
    h = x + s["scale"] * p
    mu, r = _stats(h, s["kind"])
    y = (h - mu) * r * s["w"]
    if s["b"] is not None:
        y = y + s["b"]
    return h, torch.cat((mp, rp, mu, r), 1), y


def _plain_norm(s):
    h, _, y = _norm_parts(s)
    out = {"h": h.to(s["x"].dtype)}
    if s["out"] == "mxfp8":
        rows, H = y.shape
        q, sf, _ = _quantise(y, "mxfp8")
        out["q"], out["sf"] = q.view(torch.float8_e4m3fn), sf.view(torch.float8_e8m0fnu)
    else:
        out["y"] = y.to(BF16 if s["out"] == "bf16" else torch.float32)
    return out


def _norm_grad(a, xh, r, kind):
    m1 = a.mean(-1, keepdim=True) if kind == "layer" else 0.0
    return r * (a - m1 - xh * (a * xh).mean(-1, keepdim=True))


def _col(v):
    return v.sum(0, dtype=torch.float64).float()


def _plain_norm_backward(s):
    st, kind, layer = s["stats"], s["kind"], s["kind"] == "layer"
    dy = s["dy"].float()
    xh = (s["h"].float() - st[:, 2:3]) * st[:, 3:4]
    out = {"dw": _col(dy * xh)}
    if layer:
        out["db"] = _col(dy)
    dht = s["dh"].float() + _norm_grad(dy * s["w"], xh, st[:, 3:4], kind)
    out["dx"] = dht.to(s["dx"].dtype)
    p = s["o"].float()
    if s["post"]:
        oh = (p - st[:, 0:1]) * st[:, 1:2]
        p = oh * s["wp"]
        if s["bp"] is not None:
            p = p + s["bp"]
    rows, gr = dy.shape[0], s["gate_rows"]
    dp = s["scale"] * dht
    if s["gate"] is not None:
        dg = dp * p
        if gr == 0:
            out["dgate"] = _col(dg).unsqueeze(0)
        elif gr == 1:
            out["dgate"] = dg
        else:
            n = s["gate"].shape[0]
            pad = torch.zeros((n * gr, dy.shape[1]), device=DEV)
            pad[:rows] = dg
            out["dgate"] = pad.view(n, gr, -1).sum(1, dtype=torch.float64).float()
        dp = dp * _gate_of(s, rows)
    if s["post"]:
        out["dwp"] = _col(dp * oh)
        if layer:
            out["dbp"] = _col(dp)
        dp = _norm_grad(dp * s["wp"], oh, st[:, 1:2], kind)
    out["do"] = dp.to(BF16)
    return out


# ---------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------
def run(s):
    if own:
        return _own(s)
    return {"gemm": _plain_gemm, "gemm_backward": _plain_gemm_backward, "norm": _plain_norm,
            "norm_backward": _plain_norm_backward}[s["op"]](s)


def _own(s):
    import blackhole_b200 as bh

    if s["op"] == "gemm":
        call = {"nvfp4": bh.nvfp4_bf16_gemm_fused, "mxfp4": bh.mxfp4_bf16_gemm_fused,
                "mxf8f4": bh.mxf8f4_bf16_gemm_fused}[s["fmt"]]
        call(s["M"], s["N"], s["K"], s["A"], s["SFA"], s["B"], s["SFB"], s["D"], s["alpha"],
             bias=s["bias_t"], activation=s["act"], gated=s["gated"], residual=s["res"], Z=s["Z"])
        return {"D": s["D"], "Z": s["Z"]} if s["z"] else {"D": s["D"]}
    if s["op"] == "gemm_backward":
        bh.gemm_fused_backward(s["M"], s["N"], s["dD"], s["Z"], s["dZ"], dbias=s["dbias"],
                               activation=s["act"], gated=s["gated"])
        return {"dZ": s["dZ"], "dbias": s["dbias"]}
    common = dict(kind=s["kind"], eps=1e-6, o=s["o"], post_norm=s["post"], post_weight=s["wp"],
                  post_bias=s["bp"], gate=s["gate"], gate_rows=max(0, s["gate_rows"]),
                  scale=s["scale"], weight=s["w"])
    if s["op"] == "norm":
        bh.block_norm(s["rows"], s["H"], s["x"], s["y"], h=s["h"], bias=s["b"], out_format=s["out"],
                      sf=s["sf"], **common)
        if s["out"] == "mxfp8":
            return {"h": s["h"], "q": s["y"].view(torch.float8_e4m3fn), "sf": s["sf"].view(torch.float8_e8m0fnu)}
        return {"h": s["h"], "y": s["y"]}
    bh.block_norm_backward(s["rows"], s["H"], s["h"], s["stats"], s["dx"], dy=s["dy"], dh=s["dh"],
                           do=s["do"], dweight=s["dw"], dbias=s["db"], dpost_weight=s["dwp"],
                           dpost_bias=s["dbp"], dgate=s["dgate"], **common)
    out = {"dw": s["dw"], "db": s["db"], "dx": s["dx"], "dgate": s["dgate"], "dwp": s["dwp"],
           "dbp": s["dbp"], "do": s["do"]}
    return {k: v for k, v in out.items() if v is not None}


# ---------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "gemm":
        M, N, K = c["M"], c["N"], c["K"]
        vec, a_bytes = (16, 0.5) if c["fmt"] == "nvfp4" else (32, 1.0 if c["fmt"] == "mxf8f4" else 0.5)
        n_out = N // 2 if c["gated"] else N
        return {"bytes": M * K * a_bytes + N * K * 0.5 + (M + N) * K / vec + 2 * M * n_out * (1 + c["residual"])
                + (2 * M * N if c["z"] else 0) + {"none": 0, "f32": 4, "bf16": 2}[c["bias"]] * N,
                "flops": 2.0 * M * N * K}
    if c["op"] == "gemm_backward":
        M, N = c["M"], c["N"]
        return {"bytes": 2 * M * (N // 2 if c["gated"] else N) + 4 * M * N + 4 * N, "flops": 16.0 * M * N}
    n, t = c["rows"] * c["H"], 2 if c["stream"] == "bf16" else 4
    groups = 0 if c["gate_rows"] < 0 else 1 if c["gate_rows"] == 0 else -(-c["rows"] // c["gate_rows"])
    vectors = (1 + c["post"]) * (1 + (c["kind"] == "layer"))
    if c["op"] == "norm":
        y = {"bf16": 2, "f32": 4, "mxfp8": 1 + 1 / 32}[c["out"]]
        return {"bytes": n * (2 * t + 2 + y) + 2 * groups * c["H"] + 4 * vectors * c["H"], "flops": 16.0 * n}
    return {"bytes": n * (3 * t + 2 + 2 + 2) + 16 * c["rows"] + 6 * groups * c["H"] + 8 * vectors * c["H"],
            "flops": 40.0 * n}


# ---------------------------------------------------------------------------------------
# 64 bits, from the definitions
# ---------------------------------------------------------------------------------------
def _decode64(q, sf, rows, K, fmt):
    """The operand's values from the codes' own bits, a slab of rows at a time."""
    vec = 16 if fmt == "nvfp4" else 32
    atoms = -(-K // (4 * vec))
    out = torch.empty((rows, K), dtype=torch.float64, device=DEV)
    group = torch.arange(K // vec, device=DEV)
    for r0 in range(0, rows, 1024):
        r = torch.arange(r0, min(rows, r0 + 1024), device=DEV)
        at = ((r // 128)[:, None] * atoms + (group // 4)[None]) * 512 + ((r % 32) * 16 + (r % 128) // 32 * 4)[:, None] + group % 4
        sc = sf[at].to(torch.int32)
        if fmt == "nvfp4":
            e, m = sc >> 3, (sc & 7).double()
            sc = torch.where(e == 0, m * 2.0 ** -9, torch.ldexp(1 + m / 8, e - 7))
        else:
            sc = torch.ldexp(torch.ones_like(sc, dtype=torch.float64), sc - 127)
        code = q[r].to(torch.int32)
        if fmt == "mxfp8":
            e, m = (code >> 3) & 15, (code & 7).double()
            v = torch.where(e == 0, m * 2.0 ** -9, torch.ldexp(1 + m / 8, e - 7)) * (1 - 2.0 * (code >> 7))
        else:
            code = torch.stack((code & 15, code >> 4), -1).flatten(1)
            e, m = (code >> 1) & 3, (code & 1).double()
            v = torch.where(e == 0, m / 2, torch.ldexp(1 + m / 2, e - 1)) * (1 - 2.0 * (code >> 3))
        out[r] = (v.view(len(r), -1, vec) * sc[..., None]).flatten(1)
    return out


def _act64(z, act, slope=False):
    """An activation, or its derivative, in 64 bits."""
    if act == "none":
        return torch.ones_like(z) if slope else z
    if act == "relu":
        return torch.heaviside(z, torch.zeros_like(z)) if slope else z * (z > 0)
    if act == "silu":
        t = torch.special.expit(z)
        return t + z * t * torch.special.expit(-z) if slope else z * t
    if act == "gelu":
        phi = torch.special.ndtr(z)
        return phi + z * torch.exp(-z * z / 2) / (2 * math.pi) ** 0.5 if slope else z * phi
    w = (2 / math.pi) ** 0.5 * (z + 0.044715 * z ** 3)
    t = torch.special.expit(2 * w)
    dw = (2 / math.pi) ** 0.5 * (1 + 0.134145 * z * z)
    return t + 2 * z * t * torch.special.expit(-2 * w) * dw if slope else z * t


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "gemm":
        f = case["fmt"]
        b = _decode64(s["B"], s["SFB"], s["N"], s["K"], "mxfp4" if f == "mxf8f4" else f)
        a = _decode64(s["A"], s["SFA"], s["M"], s["K"], "mxfp8" if f == "mxf8f4" else f)
        z = torch.matmul(a, b.t()).mul_(s["alpha"])
        del a, b
        if s["bias_t"] is not None:
            z += s["bias_t"].double()
        if case["gated"]:
            pair = z.view(s["M"], -1, 2)
            d = _act64(pair[..., 0], case["act"]) * pair[..., 1]
        else:
            d = _act64(z, case["act"])
        if s["res"] is not None:
            d = d + s["res"].double()
        return {"D": d, "Z": z} if case["z"] else {"D": d}
    if op == "gemm_backward":
        out_z = torch.empty(s["Z"].shape, dtype=torch.float64, device=DEV)
        for r in range(0, s["M"], 1024):
            z, d = s["Z"][r:r + 1024].double(), s["dD"][r:r + 1024].double()
            if case["gated"]:
                out_z[r:r + 1024, 0::2] = d * z[:, 1::2] * _act64(z[:, 0::2], case["act"], True)
                out_z[r:r + 1024, 1::2] = d * _act64(z[:, 0::2], case["act"])
            else:
                out_z[r:r + 1024] = d * _act64(z, case["act"], True)
        return {"dZ": out_z, "dbias": out_z.sum(0)}
    rows, H, layer = s["rows"], s["H"], s["kind"] == "layer"
    which = torch.arange(rows, device=DEV)
    which = which // s["gate_rows"] if s["gate_rows"] > 0 else which * 0
    if op == "norm":
        keep, ys = [], []
        for r in range(0, rows, 2048):
            sl = slice(r, min(rows, r + 2048))
            p = s["o"][sl].double()
            if s["post"]:
                var, mu = torch.var_mean(p, -1, correction=0, keepdim=True)
                p = (p - mu) / (var + 1e-6).sqrt() if layer else p / (p.pow(2).mean(-1, True) + 1e-6).sqrt()
                p = p * s["wp"].double() + (s["bp"].double() if layer else 0.0)
            if s["gate"] is not None:
                p = p * s["gate"].double()[which[sl]]
            h = s["x"][sl].double() + s["scale"] * p
            var, mu = torch.var_mean(h, -1, correction=0, keepdim=True)
            y = (h - mu) / (var + 1e-6).sqrt() if layer else h / (h.pow(2).mean(-1, True) + 1e-6).sqrt()
            keep.append(h)
            ys.append(y * s["w"].double() + (s["b"].double() if layer else 0.0))
        # codes next to a rounding border go either way in 32 bits: no 64-bit value for those
        y = torch.cat(ys)
        return {"h": torch.cat(keep), "q": None, "sf": None} if s["out"] == "mxfp8" else {"h": torch.cat(keep), "y": y}
    zero = lambda on, *n: torch.zeros(*n, dtype=torch.float64, device=DEV) if on else None  # noqa: E731
    post, gated = s["post"], s["gate"] is not None
    dx = torch.empty((rows, H), dtype=torch.float64, device=DEV)
    do = torch.empty_like(dx)
    dw, db, dwp, dbp = zero(True, H), zero(layer, H), zero(post, H), zero(post and layer, H)
    dgate = zero(gated, *s["gate"].shape) if gated else None
    for r in range(0, rows, 2048):
        sl = slice(r, min(rows, r + 2048))
        mp, rp, mu, rs = s["stats"][sl].double().unbind(1)
        dy, xn = s["dy"][sl].double(), (s["h"][sl].double() - mu[:, None]) * rs[:, None]
        dw += torch.einsum("rh,rh->h", dy, xn)
        if layer:
            db += dy.sum(0)
        t = dy * s["w"].double()
        along = torch.einsum("rh,rh->r", t, xn)[:, None] / H
        d = s["dh"][sl].double() + rs[:, None] * (t - (t.mean(1, True) if layer else 0.0) - xn * along)
        dx[sl] = d
        d = d * s["scale"]
        on = s["o"][sl].double()
        if post:
            on = (on - mp[:, None]) * rp[:, None]
        if gated:
            p = on * s["wp"].double() + (s["bp"].double() if layer else 0.0) if post else on
            dgate.index_add_(0, which[sl], d * p)
            d = d * s["gate"].double()[which[sl]]
        if post:
            dwp += torch.einsum("rh,rh->h", d, on)
            if layer:
                dbp += d.sum(0)
            d = d * s["wp"].double()
            along = torch.einsum("rh,rh->r", d, on)[:, None] / H
            d = rp[:, None] * (d - (d.mean(1, True) if layer else 0.0) - on * along)
        do[sl] = d
    out = {"dw": dw, "db": db, "dx": dx, "dgate": dgate, "dwp": dwp, "dbp": dbp, "do": do}
    return {k: v for k, v in out.items() if v is not None}
