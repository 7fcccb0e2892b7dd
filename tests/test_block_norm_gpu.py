"""Block norms (RMS / layer, before and after a block, gate and residual scale) on the GPU against
a plain 64-bit implementation: values, statistics, quantised operands, gradients."""
import pytest

torch = pytest.importorskip("torch")

import blackhole_b200 as bh  # noqa: E402
from tests import block_norm_cases as C  # noqa: E402

pytestmark = pytest.mark.gpu


def call(c, out_format="bf16", want_h=True, **over):
    rows, H = c["rows"], c["H"]
    T = {"bf16": torch.bfloat16, "f32": torch.float32}.get(out_format, torch.uint8)
    width = H // 2 if out_format in ("nvfp4", "mxfp4") else H
    fill = 0xAB if T == torch.uint8 else float("nan")
    r = {"out": torch.full((rows, width), fill, dtype=T, device="cuda"),
         "h": torch.full_like(c["x"], float("nan")) if c["o"] is not None and want_h else None,
         "stats": torch.full((rows, 4), float("nan"), device="cuda"), "sf": None}
    if T == torch.uint8:
        size = bh.sf_storage_bytes(rows, H) if out_format == "nvfp4" else bh.mxfp4_sf_storage_bytes(rows, H)
        r["sf"] = torch.full((size,), 0xCD, dtype=torch.uint8, device="cuda")
    kw = dict(weight=c["weight"], bias=c["bias"], kind=c["kind"], eps=c["eps"], o=c["o"],
              post_norm=c["post"], post_weight=c["post_weight"], post_bias=c["post_bias"],
              gate=c["gate"], gate_rows=c["gate_rows"], scale=c["scale"], out_format=out_format, **r)
    kw.update(over)
    bh.block_norm(rows, H, c["x"], **kw)
    torch.cuda.synchronize()
    return r


def check_forward(c, r):
    ref = C.forward64(c)
    if r["h"] is not None:
        C.close(r["h"], ref["h"], ref["mag_h"], what="h")
    C.close(r["out"], ref["y"], ref["mag_y"], what="y")
    st, want = r["stats"].cpu().double(), ref["stats"]
    # 1 / sqrt: relative; means: units of the row's mean magnitude
    assert ((st[:, 1::2] - want[:, 1::2]).abs() <= C.UNITS * C.U * (1 + ref["mag_h"].square().mean(1, keepdim=True).sqrt() * want[:, 3:]) * want[:, 1::2].abs()).all()
    m = torch.stack(((C.d(c["o"]).abs().mean(1) if c["o"] is not None else torch.zeros(c["rows"])), ref["mag_h"].mean(1)), 1)
    assert ((st[:, 0::2] - want[:, 0::2]).abs() <= C.UNITS * C.U * m + 1e-30).all()


SIZES = [(1, 8), (1, 8192), (2, 264), (3, 520), (5, 1000), (7, 4104), (2, 8200), (3, 16384), (130, 768),
         (2500, 64)]


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("stream", ["bf16", "f32"])
@pytest.mark.parametrize("rows,H", SIZES)
def test_pre_norm_of_residual(rows, H, stream, kind):
    c = C.make(rows, H, kind, stream, post=False, gate="one", seed=rows + H)
    check_forward(c, call(c, "f32" if stream == "f32" else "bf16"))


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("gate", ["none", "one", "each", 3, 64])
@pytest.mark.parametrize("rows,H", [(1, 8), (7, 1000), (129, 256), (4, 16384)])
def test_post_norm_gate_and_scale(rows, H, gate, kind):
    c = C.make(rows, H, kind, "f32" if H == 1000 else "bf16", post=True, gate=gate, seed=H,
               params="bf16" if H == 256 else "f32")
    check_forward(c, call(c, "f32"))


def test_norm_alone_without_parameters():
    c = C.make(33, 512, "layer", "bf16", with_o=False, affine=False)
    check_forward(c, call(c, "f32"))


def test_layer_norm_far_from_zero():
    """A mean a thousand times the spread: the variance is taken about the mean."""
    c = C.make(4, 2048, "layer", "f32", mean=1000.0, gate="none", seed=5)
    check_forward(c, call(c, "f32"))


def test_stream_updated_in_place_and_h_only():
    c = C.make(9, 1024, "rms", "bf16", post=True, gate="one", seed=3)
    ref = C.forward64(c)
    x = c["x"].clone()
    out = torch.empty((9, 1024), dtype=torch.bfloat16, device="cuda")
    kw = dict(weight=c["weight"], bias=c["bias"], eps=c["eps"], o=c["o"], post_norm=True, scale=c["scale"],
              post_weight=c["post_weight"], post_bias=c["post_bias"], gate=c["gate"])
    bh.block_norm(9, 1024, x, out, h=x, **kw)
    C.close(out, ref["y"], ref["mag_y"])
    C.close(x, ref["h"], ref["mag_h"])
    h = torch.empty_like(x)
    kw.update(weight=None, bias=None)
    bh.block_norm(9, 1024, c["x"], None, h=h, **kw)     # the last block: no norm follows
    assert torch.equal(h, x)


@pytest.mark.parametrize("fmt,rows,H", [(f, r, h) for f in ("nvfp4", "mxfp4", "mxfp8")
                                        for r, h in ((1, 32), (5, 1056), (130, 992), (128, 8192), (2, 8224),
                                                     (300, 96))])
def test_quantised_result_is_the_quantisers(fmt, rows, H):
    """Codes, scale factors and padding equal the framework's quantiser on the FP32 result, bit
    for bit."""
    c = C.make(rows, H, "rms", "bf16", post=True, gate="one", seed=rows * 7 + H)
    y = call(c, "f32")["out"]
    if fmt == "nvfp4":
        q, sf, scales = bh.quantize_tensor(y)
        r = call(c, fmt, global_scale=float(scales[1]))
    else:
        q, sf = (bh.quantize_tensor_mxfp4 if fmt == "mxfp4" else bh.quantize_tensor_mxfp8)(y)
        r = call(c, fmt)
    assert torch.equal(r["out"], q) and torch.equal(r["sf"], sf)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), 0.0, 3e38])
def test_rows_do_not_meet(value):
    """A row of NaN, infinities, zeros or overflowing squares leaves the other rows as they were."""
    c = C.make(6, 768, "rms", "f32", gate="none", seed=1)
    clean = call(c, "f32")["out"]
    c["x"][2] = value
    c["o"][2] = 0
    got = call(c, "f32")["out"]
    keep = [0, 1, 3, 4, 5]
    assert torch.equal(got[keep], clean[keep])
    if value == 0.0:                       # 0 / sqrt(0 + eps) * w + b
        assert torch.equal(got[2], c["bias"])


def test_rows_behind_the_last_are_left_alone():
    c = C.make(5, 256, "rms", "bf16", gate="one")
    big = torch.full((8, 256), 7.0, dtype=torch.bfloat16, device="cuda")
    bh.block_norm(5, 256, c["x"], big, weight=c["weight"], o=c["o"], gate=c["gate"])
    assert (big[5:] == 7.0).all() and (big[:5] != 7.0).any()


def backward(c, h, stats, dy, dh, in_place=False, **over):
    rows, H = c["rows"], c["H"]
    layer = c["kind"] == "layer"
    f = lambda on, *n: torch.full(n, float("nan"), device="cuda") if on else None  # noqa: E731
    r = {"dx": torch.full_like(c["x"], float("nan")), "dweight": f(dy is not None, H), "dbias": f(layer, H),
         "do": torch.full_like(c["o"], float("nan")) if c["o"] is not None else None,
         "dpost_weight": f(c["post"], H), "dpost_bias": f(c["post"] and layer, H),
         "dgate": f(c["gate"] is not None, *(c["gate"].shape if c["gate"] is not None else (1,)))}
    if in_place:
        r["dx"] = dh
    kw = dict(kind=c["kind"], weight=c["weight"], bias=c["bias"], o=c["o"], post_norm=c["post"],
              post_weight=c["post_weight"], post_bias=c["post_bias"], gate=c["gate"],
              gate_rows=c["gate_rows"], scale=c["scale"], dy=dy, dh=dh, **r)
    kw.update(over)
    bh.block_norm_backward(rows, H, h, stats, **kw)
    torch.cuda.synchronize()
    return r


def check_backward(c, r, ref):
    for k, v in r.items():
        if v is None:
            continue
        units = C.UNITS if k in ("dx", "do") else C.sum_units(c["rows"])
        if k == "dbias" and "dbias" not in ref:
            assert not v.any()
            continue
        C.close(v, ref[k], ref["mag_" + k], units=units, what=k)


def both(c, **kw):
    f = call(c, "bf16")
    h = f["h"] if f["h"] is not None else c["x"]
    r = backward(c, h, f["stats"], c["dy"], c["dh"], **kw)
    return f, h, r


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("gate", ["none", "one", "each", 3, 64])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("rows,H,stream", [(1, 8, "bf16"), (7, 1000, "f32"), (300, 256, "bf16"),
                                           (3, 16384, "bf16"), (450, 2048, "f32")])
def test_gradients(rows, H, stream, post, gate, kind):
    c = C.make(rows, H, kind, stream, post=post, gate=gate, seed=rows + H)
    f, h, r = both(c)
    check_backward(c, r, C.backward64(c, h, f["stats"], c["dy"], c["dh"]))


@pytest.mark.parametrize("rows,H,stream,gate", [(40, 640, "bf16", "one"), (5, 12296, "f32", 2), (700, 96, "f32", "each")])
def test_rms_norms_with_biases(rows, H, stream, gate):
    """RMS norms with both biases, their gradients, and types that differ: parameters BF16, gate BF16
    beside an FP32 stream."""
    c = C.make(rows, H, "rms", stream, post=True, gate=gate, params="bf16", seed=H)
    c["gate"] = c["gate"].to(torch.bfloat16)
    check_forward(c, call(c, "f32"))
    f = call(c, "bf16")
    db, dpb = (torch.full((H,), float("nan"), device="cuda") for _ in range(2))
    r = backward(c, f["h"], f["stats"], c["dy"], c["dh"], dbias=db, dpost_bias=dpb)
    r.update(dbias=db, dpost_bias=dpb)
    check_backward(c, r, C.backward64(c, f["h"], f["stats"], c["dy"], c["dh"]))


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("H,stream", [(16384, "f32"), (8200, "bf16")])
def test_rows_wider_than_one_cta(H, stream, kind):
    """Clusters of two CTAs over many rows, several rows per cluster."""
    c = C.make(170, H, kind, stream, post=True, gate=60, seed=H)
    check_forward(c, call(c, "bf16"))
    f, h, r = both(c)
    check_backward(c, r, C.backward64(c, h, f["stats"], c["dy"], c["dh"]))


def test_statistics_alone_and_gradients_of_one_side():
    """stats without out; no dy, a gate group crossing teams; no eps."""
    c = C.make(500, 256, "layer", "bf16", post=True, gate=33, seed=12)
    c["eps"] = 0.0
    ref = C.forward64(c)
    st = torch.empty((500, 4), device="cuda")
    h = torch.empty_like(c["x"])
    bh.block_norm(500, 256, c["x"], None, kind="layer", eps=0.0, o=c["o"], post_norm=True,
                  post_weight=c["post_weight"], post_bias=c["post_bias"], gate=c["gate"], gate_rows=33,
                  scale=c["scale"], h=h, stats=st)
    full = call(c, "bf16")
    assert torch.equal(st, full["stats"]) and torch.equal(h, full["h"])
    C.close(h, ref["h"], ref["mag_h"])
    check_backward(c, backward(c, h, st, None, c["dh"]), C.backward64(c, h, st, None, c["dh"]))


@pytest.mark.parametrize("rows", [5000, 9473])
@pytest.mark.parametrize("gate", ["one", 37, 700])
def test_gradients_many_rows(rows, gate):
    """Column sums over many teams; gate groups inside, across and over several teams."""
    c = C.make(rows, 512, "rms", "bf16", post=True, gate=gate, seed=rows)
    f, h, r = both(c)
    check_backward(c, r, C.backward64(c, h, f["stats"], c["dy"], c["dh"]))
    again = backward(c, h, f["stats"], c["dy"], c["dh"])
    for k in r:
        assert r[k] is None or torch.equal(r[k], again[k]), k


def test_gradients_without_block_or_one_of_the_gradients():
    c = C.make(40, 640, "layer", "bf16", with_o=False)
    f, h, r = both(c)
    check_backward(c, r, C.backward64(c, h, f["stats"], c["dy"], c["dh"]))
    c = C.make(40, 640, "rms", "bf16", post=True, gate="one")
    f = call(c)
    for dy, dh in ((c["dy"], None), (None, c["dh"])):
        check_backward(c, backward(c, f["h"], f["stats"], dy, dh), C.backward64(c, f["h"], f["stats"], dy, dh))
    dh = c["dh"].clone()
    check_backward(c, backward(c, f["h"], f["stats"], c["dy"], dh, in_place=True),
                   C.backward64(c, f["h"], f["stats"], c["dy"], c["dh"]))


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_gradients_against_differences(kind):
    """Directional derivatives of the 64-bit forward against the kernel's gradients."""
    c = C.make(6, 264, kind, "f32", post=True, gate=3, seed=9)
    f, h, r = both(c)
    dy, dh = C.d(c["dy"]), C.d(c["dh"])

    def loss(over):
        ref = C.forward64({**c, **over})
        return (ref["y"] * dy).sum() + (ref["h"] * dh).sum()

    names = {"x": "dx", "o": "do", "gate": "dgate", "weight": "dweight", "post_weight": "dpost_weight"}
    if kind == "layer":
        names.update(bias="dbias", post_bias="dpost_bias")
    gen = torch.Generator().manual_seed(4)
    for name, grad in names.items():
        v = torch.randn(c[name].shape, generator=gen, dtype=torch.float64)
        base, step = C.d(c[name]), 1e-4
        diff = (loss({name: base + step * v}) - loss({name: base - step * v})) / (2 * step)
        g = C.d(r[grad])
        # central differences: step^2 times third derivatives (values of order 1 to 30 here);
        # the gradient: half a BF16 step for do, else FP32 units of its terms
        half = torch.finfo(r[grad].dtype).eps / 2
        ref = C.backward64(c, h, f["stats"], c["dy"], c["dh"])
        tol = (half * (g * v).abs().sum() + C.sum_units(6) * C.U * (ref["mag_" + grad] * v.abs()).sum()
               + 1e3 * step * step * v.abs().sum())
        assert abs(diff - (g * v).sum()) <= tol, name


def test_own_workspace_and_streams():
    c = C.make(700, 512, "rms", "bf16", post=True, gate="one", seed=2)
    f, h, r = both(c)
    s = torch.cuda.Stream()
    size = bh.block_norm_backward_workspace_bytes(700, 512, True, 0)
    ws = torch.full((size,), 0xFF, dtype=torch.uint8, device="cuda")     # contents do not matter
    torch.cuda.synchronize()
    got = backward(c, h, f["stats"], c["dy"], c["dh"], workspace=ws, stream=s)
    for k in r:
        assert r[k] is None or torch.equal(r[k], got[k]), k


def test_captured_and_replayed():
    """Forward to MXFP8 and backward in one graph; new inputs before each replay."""
    c = C.make(260, 768, "layer", "bf16", post=True, gate=100, seed=8)
    f, h, r = both(c)
    q = call(c, "mxfp8")
    g = torch.cuda.CUDAGraph()
    st = torch.cuda.Stream()
    kw = dict(kind="layer", eps=c["eps"], o=c["o"], post_norm=True, post_weight=c["post_weight"],
              post_bias=c["post_bias"], gate=c["gate"], gate_rows=100, scale=c["scale"], weight=c["weight"])
    with torch.cuda.graph(g, stream=st):
        bh.block_norm(260, 768, c["x"], q["out"], bias=c["bias"], h=f["h"], stats=f["stats"], sf=q["sf"],
                      out_format="mxfp8", **kw)
        bh.block_norm_backward(260, 768, f["h"], f["stats"], r["dx"], dy=c["dy"], dh=c["dh"], do=r["do"],
                               dweight=r["dweight"], dbias=r["dbias"], dpost_weight=r["dpost_weight"],
                               dpost_bias=r["dpost_bias"], dgate=r["dgate"], **kw)
    for seed in (11, 12):
        new = C.make(260, 768, "layer", "bf16", post=True, gate=100, seed=seed)
        for k in ("x", "o", "gate", "weight", "bias", "post_weight", "post_bias", "dy", "dh"):
            c[k].copy_(new[k])
        g.replay()
        torch.cuda.synchronize()
        F, H, R = both(new)
        Q = call(new, "mxfp8")
        assert torch.equal(q["out"], Q["out"]) and torch.equal(q["sf"], Q["sf"])
        for k in R:
            assert torch.equal(R[k], r[k]), k


def test_offsets_past_32_bits():
    """2^31 elements and more: the last rows equal the same rows in a call of their own."""
    rows, H, tail = (1 << 18) + 3, 8192, 3
    c = C.make(tail, H, "rms", "bf16", post=True, gate="one", seed=6)
    x, o = (torch.zeros((rows, H), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    x[-tail:], o[-tail:] = c["x"], c["o"]
    h, q = torch.empty_like(x), torch.empty((rows, H), dtype=torch.uint8, device="cuda")
    sf = torch.empty(bh.mxfp4_sf_storage_bytes(rows, H), dtype=torch.uint8, device="cuda")
    st = torch.empty((rows, 4), device="cuda")
    kw = dict(weight=c["weight"], post_norm=True, post_weight=c["post_weight"], gate=c["gate"], scale=c["scale"],
              eps=c["eps"])
    bh.block_norm(rows, H, x, q, o=o, h=h, stats=st, sf=sf, out_format="mxfp8", **kw)
    small = call({**c, "bias": None, "post_bias": None}, "mxfp8")
    assert torch.equal(q[-tail:], small["out"]) and torch.equal(h[-tail:], small["h"])
    assert torch.equal(sf[-small["sf"].numel():], small["sf"]) and not q[:-tail].any()
    del q, sf
    dx, do = x, o                                  # written over what the backward pass does not read
    dy, dh = (torch.zeros((rows, H), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    dy[-tail:], dh[-tail:] = c["dy"], c["dh"]
    o2 = torch.zeros_like(o)
    o2[-tail:] = c["o"]
    dw, dg = torch.empty(H, device="cuda"), torch.empty((1, H), device="cuda")
    bh.block_norm_backward(rows, H, h, st, dx, dy=dy, dh=dh, o=o2, do=do, dweight=dw, dgate=dg, **kw)
    ref = C.backward64({**c, "bias": None, "post_bias": None}, h[-tail:], st[-tail:], c["dy"], c["dh"])
    C.close(dx[-tail:], ref["dx"], ref["mag_dx"])
    C.close(do[-tail:], ref["do"], ref["mag_do"])
    C.close(dw, ref["dweight"], ref["mag_dweight"], units=C.sum_units(rows))
    C.close(dg, ref["dgate"], ref["mag_dgate"], units=C.sum_units(rows))


def test_several_threads_and_streams():
    """Three host threads, each with its own stream and sizes, forward and backward at once."""
    import threading
    cases = [C.make(r, h, k, "bf16", post=True, gate=g, seed=r)
             for r, h, k, g in ((300, 1024, "rms", "one"), (77, 4104, "layer", 11), (900, 512, "rms", "each"))]
    want = [both(c) for c in cases]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        c, (f, h, r) = cases[i], want[i]
        s = torch.cuda.Stream()
        try:
            with torch.cuda.stream(s):
                for _ in range(5):
                    F = call(c, "bf16")
                    R = backward(c, F["h"], F["stats"], c["dy"], c["dh"])
                    s.synchronize()
                    if not torch.equal(F["out"], f["out"]) or any(
                            r[k] is not None and not torch.equal(r[k], R[k]) for k in r):
                        bad.append(i)
        except Exception as e:          # an exception in a thread is a failure too
            bad.append((i, repr(e)))

    ts = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not bad


def test_tensors_that_do_not_fit():
    c = C.make(4, 256, "rms", "bf16", gate="one")
    ok = dict(weight=c["weight"], o=c["o"], gate=c["gate"])
    out = torch.empty((4, 256), dtype=torch.bfloat16, device="cuda")
    bh.block_norm(4, 256, c["x"], out, **ok)
    for over in (dict(o=c["o"].float()), dict(o=c["o"][:3]), dict(weight=c["weight"][:128]), dict(weight=c["weight"].half()),
                 dict(bias=torch.zeros(256, dtype=torch.bfloat16, device="cuda")), dict(h=c["x"].float()),
                 dict(gate=c["gate"].cpu()), dict(gate=c["gate"], gate_rows=2), dict(stats=torch.empty(4, 3, device="cuda")),
                 dict(o=torch.zeros((256, 4), dtype=torch.bfloat16, device="cuda").T)):
        with pytest.raises(ValueError):
            bh.block_norm(4, 256, c["x"], out, **{**ok, **over})
    with pytest.raises(ValueError):
        bh.block_norm(4, 256, c["x"], torch.empty((4, 256), dtype=torch.uint8, device="cuda"), out_format="mxfp8",
                      sf=torch.empty(8, dtype=torch.uint8, device="cuda"), **ok)
    with pytest.raises(bh.BlackholeError):       # a workspace that is too small
        both(c, workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
