"""Products with bias, activation or gated activation and residual in their epilogue, and the
gradient through it, on the GPU against a plain 64-bit implementation."""
import pytest

torch = pytest.importorskip("torch")

import blackhole_b200 as bh  # noqa: E402
from tests import block_norm_cases as NC  # noqa: E402
from tests import gemm_fused_cases as C  # noqa: E402

pytestmark = pytest.mark.gpu

EPILOGUES = [  # act, gated, bias, residual, Z
    ("none", False, "bf16", True, False), ("none", False, None, True, True), ("relu", False, "f32", False, True),
    ("gelu", False, "bf16", True, True), ("gelu_tanh", False, "f32", True, False), ("silu", False, None, False, False),
    ("silu", True, None, False, False), ("gelu", True, "bf16", True, True), ("relu", True, "f32", True, False),
    ("none", True, "f32", False, True), ("gelu_tanh", True, None, True, True)]


@pytest.mark.parametrize("act,gated,bias,residual,z", EPILOGUES)
@pytest.mark.parametrize("fmt", C.FMTS)
@pytest.mark.parametrize("M,N,K", [(1, 256, 256), (16, 1040, 512), (100, 400, 384), (300, 528, 640)])
def test_against_64_bits(M, N, K, fmt, act, gated, bias, residual, z):
    c = C.make(fmt, M, N, K, act, gated, bias, residual, z, beta=0.5, seed=M)
    C.call(c)
    C.check(c)


@pytest.mark.parametrize("schedule", ["1sm", "2sm", "skinny", "skinny_noprefetch"])
@pytest.mark.parametrize("fmt", C.FMTS)
@pytest.mark.parametrize("M,N,K,gated", [(1, 16, 128, True), (3, 8, 256, False), (33, 2064, 1152, True),
                                         (128, 136, 2048, False), (70, 4096, 4096, True)])
def test_every_schedule(M, N, K, gated, fmt, schedule):
    c = C.make(fmt, M, N, K, "silu", gated, "bf16", True, True, beta=-1.25, seed=N)
    C.call(c, schedule=schedule)
    C.check(c)


@pytest.mark.parametrize("fmt,M,N,K", [("nvfp4", 7, 24, 32), ("nvfp4", 257, 264, 288), ("mxfp4", 511, 776, 96),
                                       ("nvfp4", 640, 2048, 4096)])
def test_tails(fmt, M, N, K):
    """K tails, ragged tiles, more tiles than one wave's share of an SM."""
    c = C.make(fmt, M, N, K, "gelu_tanh", False, "f32", True, True, seed=3)
    C.call(c)
    C.check(c)


@pytest.mark.parametrize("fmt", C.FMTS)
@pytest.mark.parametrize("M", [1, 16, 64, 200, 384])
def test_empty_epilogue_is_the_plain_product(fmt, M):
    """No bias, activation or residual: bit for bit the plain call's D."""
    c = C.make(fmt, M, 640, 1024, seed=M)
    C.call(c)
    plain = torch.empty_like(c["D"])
    args = (M, 640, 1024, c["A"], c["SFA"], c["B"], c["SFB"], plain, c["alpha"])
    (bh.nvfp4_bf16_gemm if fmt == "nvfp4" else bh.mxfp4_bf16_gemm if fmt == "mxfp4" else bh.mxf8f4_bf16_gemm)(*args)
    torch.cuda.synchronize()
    assert torch.equal(plain.view(torch.int16), c["D"].view(torch.int16))


@pytest.mark.parametrize("M", [5, 130, 700])
@pytest.mark.parametrize("gated", [False, True])
def test_residual_updated_in_place_and_rows_behind(M, gated):
    c = C.make("nvfp4", M, 512, 512, "silu", gated, "bf16", True, seed=9)
    n_out = c["D"].shape[1]
    big = torch.full((M + 40, n_out), 3.0, dtype=torch.bfloat16, device="cuda")
    big[:M] = c["residual"]
    C.call(c, D=big, residual=big)
    torch.cuda.synchronize()
    c["D"] = big[:M]
    assert (big[M:] == 3.0).all()
    C.check(c)


def test_schedule_refusals_and_missing_workspace():
    c = C.make("nvfp4", 129, 256, 256, seed=1)
    for kw in (dict(schedule="skinny"), ):
        with pytest.raises(bh.BlackholeError):
            C.call(c, **kw)
    c = C.make("nvfp4", 16, 256, 256, seed=1)
    small = torch.zeros(64, dtype=torch.uint8, device="cuda")
    with pytest.raises(bh.BlackholeError):
        C.call(c, workspace=small)
    with pytest.raises(ValueError):
        C.call(c, D=c["D"].float())
    with pytest.raises(ValueError):
        C.call(c, D=c["D"][:8])
    for k in ("A", "SFA", "B", "SFB"):
        with pytest.raises(ValueError):
            C.call({**c, k: c[k][:-1]})


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("M", [4, 300])
def test_tails_of_the_activations(M, act):
    """Biases from -80 to 80: far negative values keep their relative accuracy, nothing overflows."""
    c = C.make("nvfp4", M, 256, 64, act, bias="f32", seed=1)
    c["bias"] = torch.linspace(-80, 80, 256).cuda()
    C.call(c)
    C.check(c)


def test_non_finite_bias_and_residual_stay_in_their_columns():
    for M in (8, 200, 400):
        c = C.make("nvfp4", M, 256, 256, "silu", bias="f32", residual=True, seed=2)
        C.call(c)
        clean = c["D"].clone()
        c["bias"][17], c["residual"][3, 40] = float("nan"), float("inf")
        C.call(c)
        torch.cuda.synchronize()
        assert torch.isnan(c["D"][:, 17]).all() and c["D"][3, 40] == float("inf")
        same = torch.ones_like(clean, dtype=torch.bool)
        same[:, 17], same[3, 40] = False, False
        assert torch.equal(c["D"][same], clean[same])


def test_captured_and_replayed_with_own_workspaces():
    """Two captured decode products with workspaces of their own, replayed on two streams."""
    cases = [C.make("mxf8f4", 16, 1024, 2048, "silu", True, "bf16", True, seed=s) for s in (1, 2)]
    size = bh.workspace_bytes(16, 1024, 2048)
    graphs = []
    for c in cases:
        ws = torch.zeros(size, dtype=torch.uint8, device="cuda")
        C.call(c, workspace=ws)
        torch.cuda.synchronize()
        c["want"] = c["D"].clone()
        g, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(g, stream=st):
            C.call(c, workspace=ws)
        graphs.append((g, st, c, ws))
        c["D"].fill_(float("nan"))
    torch.cuda.synchronize()
    for _ in range(5):
        for g, st, c, _ws in graphs:
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for g, st, c, _ws in graphs:
        assert torch.equal(c["D"], c["want"])
        C.check(c)


def epilogue_grads(M, N, act, gated, seed=0):
    g = torch.Generator().manual_seed(seed)
    Z = (torch.randn(M, N, generator=g) * 2).to(torch.bfloat16)
    dD = torch.randn(M, N // 2 if gated else N, generator=g).to(torch.bfloat16)
    z, d = Z.double(), dD.double()
    if gated:
        zg, zu = z[:, 0::2], z[:, 1::2]
        ref = torch.stack((d * zu * C.slope64(zg, act), d * C.act64(zg, act)), -1).flatten(1)
        mag = torch.stack((d.abs() * zu.abs(), d.abs() * zg.abs()), -1).flatten(1)
        units = C.act_units(zg, act).repeat_interleave(2, 1)
    else:
        ref, mag, units = d * C.slope64(z, act), d.abs(), C.act_units(z, act)
    # slopes are sums of terms of at most (1 + |z|) magnitude each
    err = C.U * (units + 4) * mag * (2 + (z[:, 0::2].abs().repeat_interleave(2, 1) if gated else z.abs()))
    return Z.cuda(), dD.cuda(), ref, err


@pytest.mark.parametrize("act", list(bh.ACTIVATIONS))
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("M,N", [(1, 16), (7, 1008), (333, 256), (1024, 528), (1025, 304), (5000, 272)])
def test_gradient_through_the_epilogue(M, N, gated, act):
    Z, dD, ref, err = epilogue_grads(M, N, act, gated, M)
    dZ = torch.full((M, N), float("nan"), dtype=torch.bfloat16, device="cuda")
    db = torch.full((N,), float("nan"), device="cuda")
    bh.gemm_fused_backward(M, N, dD, Z, dZ, dbias=db, activation=act, gated=gated)
    torch.cuda.synchronize()
    C.within(dZ, ref, err, "dZ")
    C.within(db, ref.sum(0), err.sum(0) + C.U * (M / 8 + 64) * ref.abs().sum(0), "dbias")
    again = torch.empty_like(db)
    z2 = Z.clone()
    bh.gemm_fused_backward(M, N, dD, z2, z2, dbias=again, activation=act, gated=gated)   # over Z itself
    torch.cuda.synchronize()
    assert torch.equal(again, db) and torch.equal(z2, dZ)
    alone = torch.empty_like(dZ)
    bh.gemm_fused_backward(M, N, dD, Z, alone, activation=act, gated=gated)
    assert torch.equal(alone, dZ)


@pytest.mark.parametrize("act", list(bh.ACTIVATIONS))
@pytest.mark.parametrize("gated", [False, True])
def test_gradient_against_differences(act, gated):
    M, N = 9, 64
    Z, dD, ref, err = epilogue_grads(M, N, act, gated, 2)
    dZ = torch.empty_like(Z)
    bh.gemm_fused_backward(M, N, dD, Z, dZ, activation=act, gated=gated)
    got, z, d, step = dZ.cpu().double(), Z.cpu().double(), dD.cpu().double(), 1e-5

    def loss(v):
        return (d * (C.act64(v[:, 0::2], act) * v[:, 1::2] if gated else C.act64(v, act)))

    for j in range(N):
        e = torch.zeros(M, N, dtype=torch.float64)
        e[:, j] = step
        diff = (loss(z + e) - loss(z - e)).sum(1) / (2 * step)
        # a ReLU's kink between the two points is left out (|z| < step does not occur in BF16 draws
        # other than exact zeros)
        keep = (z[:, j & ~1 if gated else j].abs() > 2 * step)
        tol = torch.finfo(torch.bfloat16).eps / 2 * got[:, j].abs() + 2 * err[:, j] + 1e-8
        assert ((diff - got[:, j]).abs() <= tol)[keep].all(), j


def test_extreme_pre_activations():
    """Infinite-looking and huge pre-activations give the limits of the slopes, not NaN."""
    z = torch.tensor([-3e38, -1e20, -200.0, -0.0, 0.0, 200.0, 1e20, 3e38], dtype=torch.bfloat16, device="cuda").repeat(2, 1)
    d = torch.ones_like(z)
    for act in ("relu", "gelu", "gelu_tanh", "silu"):
        out = torch.empty_like(z)
        bh.gemm_fused_backward(2, 8, d, z, out, activation=act)
        want = torch.tensor([0, 0, 0, 0.5, 0.5, 1, 1, 1], device="cuda")
        if act == "relu":
            want[3:5] = 0
        assert torch.equal(out.float(), want.repeat(2, 1)), (act, out)


def test_an_mlp_block_forward_and_backward():
    """Norm to MXFP8 -> gated product -> MXFP8 -> product with residual -> norm; each stage against
    64 bits on the codes that the stage before it made, then the gradients back through them."""
    T, H, I = 200, 512, 768
    dev = "cuda"
    n = NC.make(T, H, "rms", "bf16", post=True, gate="one", seed=4)
    up = C.operands("mxf8f4", 1, 2 * I, H, seed=21)
    W1, SF1 = torch.from_numpy(up["B"]).to(dev), torch.from_numpy(up["SFB"]).to(dev)
    down = C.operands("mxf8f4", 1, H, I, seed=22)
    W2, SF2 = torch.from_numpy(down["B"]).to(dev), torch.from_numpy(down["SFB"]).to(dev)
    q = torch.empty((T, H), dtype=torch.uint8, device=dev)
    sf = torch.empty(bh.mxfp4_sf_storage_bytes(T, H), dtype=torch.uint8, device=dev)
    h, st = torch.empty_like(n["x"]), torch.empty((T, 4), device=dev)
    kw = dict(o=n["o"], post_norm=True, post_weight=n["post_weight"], gate=n["gate"], scale=n["scale"], eps=n["eps"],
              weight=n["weight"])
    bh.block_norm(T, H, n["x"], q, h=h, stats=st, sf=sf, out_format="mxfp8", **kw)
    Z = torch.empty((T, 2 * I), dtype=torch.bfloat16, device=dev)
    act = torch.empty((T, I), dtype=torch.bfloat16, device=dev)
    bh.mxf8f4_bf16_gemm_fused(T, 2 * I, H, q, sf, W1, SF1, act, activation="silu", gated=True, Z=Z)
    q2, sf2 = bh.quantize_tensor_mxfp8(act)
    out = torch.empty((T, H), dtype=torch.bfloat16, device=dev)
    bh.mxf8f4_bf16_gemm_fused(T, H, I, q2, sf2, W2, SF2, out, residual=h)
    torch.cuda.synchronize()
    assert bh.device_status(0) == 0

    def value(codes, scales, rows, K, kind):
        import numpy as np
        v, s = C.O.decode_operand(codes.cpu().numpy().ravel(), scales.cpu().numpy(), rows, K, kind)
        return torch.from_numpy(v).double() * torch.from_numpy(np.repeat(s, 32, 1)).double()

    n2 = {**n, "bias": None, "post_bias": None}
    ref = NC.forward64(n2)
    NC.close(h, ref["h"], ref["mag_h"], what="h")
    a = value(q, sf, T, H, "mxfp8")
    # an E4M3 code is off by half a step of at most 2^-4 of its value, or of the block's subnormal
    # step 2^-9 of a scale of at least amax / 512; saturation at 448 of up to 512 costs 1/8
    block = ref["y"].view(T, -1, 32).abs().amax(-1, keepdim=True).expand(-1, -1, 32).reshape(T, H)
    assert ((a - ref["y"]).abs() <= ref["y"].abs() / 16 + block * (1 / 8) + 1e-6).all()
    w1, w2 = value(W1, SF1, 2 * I, H, "mxfp4"), value(W2, SF2, H, I, "mxfp4")
    z, mag = a @ w1.T, a.abs() @ w1.abs().T
    C.within(Z, z, C.U * (H ** 0.5 + 8) * mag, "Z")
    c = {"bias": None, "N": 2 * I, "K": H, "gated": True, "act": "silu", "residual": None, "beta": 1.0,
         "ref": {"prod": z, "mag": mag}}
    _, _, u, e = C.expected(c)
    C.within(act, u, e, "act")
    b = value(q2, sf2, T, I, "mxfp8")
    prod, mag = b @ w2.T, b.abs() @ w2.abs().T
    C.within(out, prod + h.cpu().double(), C.U * (I ** 0.5 + 8) * (mag + h.cpu().double().abs()), "out")

    # backward: the residual's gradient into h, the gated activation's from Z, the norms' from h
    g = torch.Generator().manual_seed(1)
    dact = torch.randn(T, I, generator=g).to(torch.bfloat16).cuda()
    dZ = torch.empty_like(Z)
    bh.gemm_fused_backward(T, 2 * I, dact, Z, dZ, activation="silu", gated=True)
    zz, dd = Z.cpu().double(), dact.cpu().double()
    want = torch.stack((dd * zz[:, 1::2] * C.slope64(zz[:, 0::2], "silu"), dd * C.act64(zz[:, 0::2], "silu")), -1).flatten(1)
    C.within(dZ, want, C.U * 200 * (1 + zz.abs().max()) ** 2 * dd.abs().repeat_interleave(2, 1), "dZ")
    dy = (dZ.float() @ w1.float().cuda()).to(torch.bfloat16)      # the operand's gradient
    dx, do = torch.empty_like(n["x"]), torch.empty_like(n["o"])
    dw, dwp, dg = (torch.empty(H, device=dev) for _ in range(3))
    bh.block_norm_backward(T, H, h, st, dx, dy=dy, dh=n["dh"], do=do, dweight=dw, dpost_weight=dwp,
                           dgate=dg.view(1, H), **kw)
    torch.cuda.synchronize()
    r = NC.backward64(n2, h, st, dy, n["dh"])
    for name, got in (("dx", dx), ("do", do)):
        NC.close(got, r[name], r["mag_" + name], what=name)
    for name, got in (("dweight", dw), ("dpost_weight", dwp), ("dgate", dg.view(1, H))):
        NC.close(got, r[name], r["mag_" + name], units=NC.sum_units(T), what=name)


def test_offsets_past_32_bits():
    """D, Z, residual and the gradient with more than 2^31 elements: the last rows equal the same rows
    in calls of their own."""
    M, N, K, tail = 65536 + 40, 32768, 256, 40
    c = C.make("mxfp4", tail, N, K, "gelu", bias="f32", residual=True, z=True, seed=3)
    C.call(c)
    A = torch.zeros((M, K // 2), dtype=torch.uint8, device="cuda")
    A[-tail:] = c["A"].view(tail, K // 2)
    SFA = torch.full((bh.mxfp4_sf_storage_bytes(M, K),), 127, dtype=torch.uint8, device="cuda")
    SFA[-c["SFA"].numel():] = c["SFA"]                  # (65536 rows are whole 128-row blocks)
    D, Z, res = (torch.zeros((M, N), dtype=torch.bfloat16, device="cuda") for _ in range(3))
    res[-tail:] = c["residual"]
    bh.mxfp4_bf16_gemm_fused(M, N, K, A, SFA, c["B"], c["SFB"], D, c["alpha"], bias=c["bias"], activation="gelu",
                             residual=res, Z=Z)
    torch.cuda.synchronize()
    C.check(c)
    c["D"], c["Z"] = D[-tail:], Z[-tail:]
    C.check(c)
    dD, dZ = D, res
    dD[:-tail] = 0
    db = torch.empty(N, device="cuda")
    bh.gemm_fused_backward(M, N, dD, Z, dZ, dbias=db, activation="gelu")
    small, db2 = torch.empty((tail, N), dtype=torch.bfloat16, device="cuda"), torch.empty(N, device="cuda")
    bh.gemm_fused_backward(tail, N, dD[-tail:], Z[-tail:], small, dbias=db2, activation="gelu")
    assert torch.equal(dZ[-tail:], small) and not dZ[:-tail].any()
    mag = small.float().abs().sum(0)
    assert ((db - db2).abs() <= 200 * C.U * mag + 1e-30).all()


def test_several_threads_and_streams():
    """Three host threads, each with its own stream, shape and schedule, at once."""
    import threading
    cases = []
    for M, gated in ((8, True), (150, False), (520, True)):
        cases.append(C.make("nvfp4", M, 1024, 1024, "silu", gated, "bf16", True, True, seed=M))
        C.call(cases[-1])
    torch.cuda.synchronize()
    want = [c["D"].clone() for c in cases]
    bad = []

    def work(i):
        c, s = cases[i], torch.cuda.Stream()
        try:
            with torch.cuda.stream(s):
                for _ in range(10):
                    D = torch.zeros_like(want[i])
                    C.call(c, D=D)
                    s.synchronize()
                    if not torch.equal(D, want[i]):
                        bad.append(i)
        except Exception as e:
            bad.append((i, repr(e)))

    ts = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not bad and bh.device_status(0) == 0
