"""Inputs, 64-bit plain forms and error bounds for the block norm tests.

Bounds: a rounding to type t is off by at most finfo(t).eps / 2 of the value.  What the FP32
arithmetic may add is counted in units of 2^-24 of the magnitudes that meet in the result
(`mag`): a sum over a row is a tree of at most 16 + 5 + 16 additions, so a mean or a sum of
squares is off by at most 40 units and its inverse root by 20 + 2; a normed value carries its own
input's error, the mean's, the root's and 4 roundings.  Two norms in a row stay below 200 units.
"""
from __future__ import annotations

import torch

U = 2.0 ** -24
UNITS = 200.0


def make(rows, H, kind="rms", stream="bf16", post=False, gate="none", params="f32", affine=True,
         with_o=True, seed=0, mean=0.0, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, std=1.0, mu=0.0: torch.randn(*s, generator=g, dtype=torch.float64) * std + mu  # noqa: E731
    T = torch.bfloat16 if stream == "bf16" else torch.float32
    P = torch.bfloat16 if params == "bf16" else torch.float32
    c = {"rows": rows, "H": H, "kind": kind, "post": post, "scale": 0.75, "eps": 1e-5}
    c["x"] = r(rows, H, mu=mean).to(T)
    c["o"] = r(rows, H, std=0.5, mu=mean / 2).to(torch.bfloat16) if with_o else None
    c["weight"] = r(H, std=0.2, mu=1.0).to(P) if affine else None
    c["bias"] = r(H, std=0.2).to(P) if affine else None
    c["post_weight"] = r(H, std=0.2, mu=1.0).to(P) if post and affine else None
    c["post_bias"] = r(H, std=0.2).to(P) if post and affine else None
    c["gate_rows"] = {"none": 0, "one": 0, "each": 1}.get(gate, gate)
    if gate == "none" or not with_o:
        c["gate"] = None
    else:
        n = 1 if gate == "one" else -(-rows // c["gate_rows"])
        c["gate"] = r(n, H).to(torch.float32 if stream == "f32" else torch.bfloat16)
    c["dy"] = r(rows, H, std=0.3).to(torch.bfloat16)
    c["dh"] = r(rows, H, std=0.3).to(T)
    return {k: v.to(device) if isinstance(v, torch.Tensor) else v for k, v in c.items()}


def d(t):
    return None if t is None else t.detach().cpu().double()


def _norm(v, mag, kind, eps, w, b):
    mu = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[:, :1])
    rstd = ((v - mu).square().mean(-1, keepdim=True) + eps).rsqrt()
    w = torch.ones(()) if w is None else w
    b = torch.zeros(()) if b is None else b
    m = (mag + mu.abs() + (mag.mean(-1, keepdim=True) if kind == "layer" else 0)) * rstd * w.abs() + b.abs()
    # the root's error comes from the whole row's
    m = m + (v - mu).abs() * rstd * w.abs() * (mag.square().mean(-1, keepdim=True).sqrt() * rstd).clamp(min=1)
    return mu, rstd, (v - mu) * rstd * w + b, m


def gate_rows_of(c):
    if c["gate"] is None:
        return None
    at = torch.arange(c["rows"]) // c["gate_rows"] if c["gate_rows"] else torch.zeros(c["rows"], dtype=torch.long)
    return at


def forward64(c):
    """{h, y, stats} and their magnitudes, in 64 bits."""
    x = d(c["x"])
    h, mh = x, x.abs()
    zero = torch.zeros_like(x[:, :1])
    mp = rp = zero
    if c["o"] is not None:
        p, mag = d(c["o"]), d(c["o"]).abs()
        if c["post"]:
            mp, rp, p, mag = _norm(p, mag, c["kind"], c["eps"], d(c["post_weight"]), d(c["post_bias"]))
        g = d(c["gate"])[gate_rows_of(c)] if c["gate"] is not None else 1.0
        h = x + c["scale"] * g * p
        mh = x.abs() + abs(c["scale"]) * (g.abs() if torch.is_tensor(g) else g) * mag
    mu, r, y, my = _norm(h, mh, c["kind"], c["eps"], d(c["weight"]), d(c["bias"]))
    return {"h": h, "y": y, "stats": torch.cat((mp, rp, mu, r), 1), "mag_h": mh, "mag_y": my}


def backward64(c, h, stats, dy, dh):
    """Gradients from the stored h and statistics, and their magnitudes, in 64 bits."""
    h, st, layer = d(h), d(stats), c["kind"] == "layer"
    one = torch.ones(c["H"], dtype=torch.float64)
    w = one if c["weight"] is None else d(c["weight"])
    out = {}
    dht = d(dh) if dh is not None else torch.zeros_like(h)
    mag = dht.abs()

    def grad(a, n, r, m):
        v = r * (a - (a.mean(-1, keepdim=True) if layer else 0) - n * (a * n).mean(-1, keepdim=True))
        mm = r.abs() * (m + (m.mean(-1, keepdim=True) if layer else 0) + n.abs() * (m * n.abs()).mean(-1, keepdim=True))
        return v, mm

    if dy is not None:
        a = d(dy)
        n = (h - st[:, 2:3]) * st[:, 3:4]
        mn = (h.abs() + st[:, 2:3].abs()) * st[:, 3:4]
        out["dweight"], out["mag_dweight"] = (a * n).sum(0), (a.abs() * mn).sum(0)
        out["dbias"], out["mag_dbias"] = a.sum(0), a.abs().sum(0)
        v, m = grad(a * w, n, st[:, 3:4], (a * w).abs())
        m = m + st[:, 3:4] * mn * ((a * w).abs() * mn).mean(-1, keepdim=True)
        dht, mag = dht + v, mag + m
    out["dx"], out["mag_dx"] = dht, mag
    if c["o"] is None:
        return out
    o = d(c["o"])
    n, mn, pw, p = o, o.abs(), one, o
    if c["post"]:
        n = (o - st[:, 0:1]) * st[:, 1:2]
        mn = (o.abs() + st[:, 0:1].abs()) * st[:, 1:2]
        pw = one if c["post_weight"] is None else d(c["post_weight"])
        p = n * pw + (0 if c["post_bias"] is None else d(c["post_bias"]))
    mp = mn * pw.abs() + (0 if c["post_bias"] is None else d(c["post_bias"]).abs())
    dp, mag = c["scale"] * dht, abs(c["scale"]) * mag
    if c["gate"] is not None:
        at = gate_rows_of(c)
        z = torch.zeros(c["gate"].shape, dtype=torch.float64)
        out["dgate"], out["mag_dgate"] = z.index_add(0, at, dp * p), z.index_add(0, at, mag * mp)
        g = d(c["gate"])[at]
        dp, mag = dp * g, mag * g.abs()
    if c["post"]:
        out["dpost_weight"], out["mag_dpost_weight"] = (dp * n).sum(0), (mag * mn).sum(0)
        out["dpost_bias"], out["mag_dpost_bias"] = dp.sum(0), mag.sum(0)
        m1 = mag * pw.abs()
        dp, mag = grad(dp * pw, n, st[:, 1:2], m1)
        mag = mag + st[:, 1:2] * mn * (m1 * mn).mean(-1, keepdim=True)
    out["do"], out["mag_do"] = dp, mag
    return out


def close(got, ref, mag, units=UNITS, what=""):
    """|got - ref| <= half a step of got's type + `units` * 2^-24 * mag, everywhere."""
    half = 0.0 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps / 2
    if got.dtype == torch.float32:
        half = U
    got = d(got)
    tol = half * ref.abs() * (1 + units * U) + units * U * mag + 1e-37
    worst = ((got - ref).abs() / tol).max().item()
    assert torch.isfinite(got).all() and worst <= 1.0, f"{what}: {worst:.3g} times the bound"


def sum_units(rows):
    """FP32 column sums: each term carries UNITS, the additions one unit each (a CTA's rows one
    after another, then at most 32 + teams / 32 partials)."""
    return UNITS + min(rows, 2 * 148) + rows / 148 + 148 * 16 / 32 + 8
