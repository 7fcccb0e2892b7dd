"""What the fused products and their gradient refuse, before any device work (no GPU needed)."""
import pytest

import blackhole_b200 as bh
from blackhole_b200.fused import _EPILOGUE

A = 1 << 40          # aligned addresses that are never dereferenced: every case is refused first
S = 1 << 34
CALLS = [bh.nvfp4_bf16_gemm_fused, bh.mxfp4_bf16_gemm_fused, bh.mxf8f4_bf16_gemm_fused]


def forward(call, **over):
    v = dict(M=16, N=256, K=256, A=A, SFA=A + S, B=A + 2 * S, SFB=A + 3 * S, D=A + 4 * S, bias=A + 5 * S,
             residual=A + 6 * S, Z=A + 7 * S, activation="silu", gated=True, stream=0)
    v.update(over)
    pos = [v.pop(k) for k in ("M", "N", "K", "A", "SFA", "B", "SFB", "D")]
    call(*pos, **v)


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("over", [
    dict(M=0), dict(N=4), dict(N=260), dict(N=264), dict(K=16), dict(K=272), dict(A=None), dict(D=None),
    dict(SFB=A + 3 * S + 8), dict(bias=A + 5 * S + 8), dict(residual=A + 6 * S + 2), dict(Z=A + 7 * S + 4),
    dict(beta=float("nan")), dict(beta=float("inf")), dict(residual=A + 4 * S + 16), dict(Z=A + 4 * S),
    dict(Z=A + 6 * S + 16),
])
def test_forward_refusals(call, over):
    with pytest.raises(bh.BlackholeError) as e:
        forward(call, **over)
    assert e.value.code == 1


def test_format_refusals():
    with pytest.raises(bh.BlackholeError):
        forward(bh.mxf8f4_bf16_gemm_fused, K=288)
    with pytest.raises(bh.BlackholeError):
        forward(bh.mxf8f4_bf16_gemm_fused, B=A + 2 * S + 16)


def test_names_and_null_epilogue():
    for k, v in (("activation", "tanh"), ("schedule", "4sm")):
        with pytest.raises(KeyError):
            forward(CALLS[0], **{k: v})
    L = bh.load()
    for f in ("nvfp4", "mxfp4", "mxf8f4"):
        fn = getattr(L, f"blackhole_sm100_{f}_bf16_gemm_fused")
        args = (16, 256, 256, A, A + S, A + 2 * S, A + 3 * S, A + 4 * S, 1.0)
        assert fn(*args, None, 0, None, 0, None) == 1
        for sched in (-1, 5):
            assert fn(*args, _EPILOGUE.pack(0, 0, 0, 1.0, 0, 0, 0), sched, None, 0, None) == 1
        for act in (-1, 5):
            assert fn(*args, _EPILOGUE.pack(act, 0, 0, 1.0, 0, 0, 0), 0, None, 0, None) == 1


@pytest.mark.parametrize("over", [
    dict(M=0), dict(M=-4), dict(M=(1 << 30) + 1), dict(N=0), dict(N=12), dict(N=264), dict(dD=None), dict(Z=None), dict(dZ=None),
    dict(dD=A + 8), dict(Z=A + S + 2), dict(dZ=A + 2 * S + 4), dict(dbias=A + 3 * S + 8), dict(dZ=A),
    dict(dZ=A + S + 16), dict(dZ=A + 16, gated=False), dict(workspace_bytes=4, M=100000),
    dict(workspace=A + 4 * S + 8),
])
def test_backward_refusals(over):
    v = dict(M=5000, N=256, dD=A, Z=A + S, dZ=A + 2 * S, dbias=A + 3 * S, workspace=A + 4 * S,
             workspace_bytes=1 << 30, activation="silu", gated=True, stream=0)
    v.update(over)
    pos = [v.pop(k) for k in ("M", "N", "dD", "Z", "dZ")]
    with pytest.raises(bh.BlackholeError) as e:
        bh.gemm_fused_backward(*pos, **v)
    assert e.value.code == 1


def test_backward_unknown_activation():
    L = bh.load()
    for act in (-1, 5):
        assert L.blackhole_sm100_gemm_fused_backward(8, 256, A, A + S, A + 2 * S, None, act, 0, None, 0, None) == 1


@pytest.mark.parametrize("M,N", [(1, 8), (8, 256), (333, 1000), (16384, 28672), (100000, 8)])
def test_backward_workspace_size(M, N):
    n = bh.gemm_fused_backward_workspace_bytes(M, N)
    assert n % (4 * N) == 0 and 0 <= n // (4 * N) <= 148 * 8
    for bad in ((0, N), (M, 12), (M, 0)):
        assert bh.gemm_fused_backward_workspace_bytes(*bad) < 0


def test_tensors_are_checked():
    torch = pytest.importorskip("torch")
    with pytest.raises(ValueError):
        forward(CALLS[0], D=torch.zeros(16, 128, dtype=torch.bfloat16))       # not on a GPU
    with pytest.raises(TypeError):
        forward(CALLS[0], bias=[0.0] * 256)


def test_numpy_numbers_are_taken():
    import numpy as np
    for call in CALLS:
        with pytest.raises(bh.BlackholeError):                       # refused by the library, not by ctypes
            forward(call, M=np.int64(0), N=np.int32(256), K=np.int64(256), alpha=np.float32(0.5), beta=np.float32(1))
    with pytest.raises(bh.BlackholeError):
        bh.gemm_fused_backward(np.int64(0), np.int64(256), A, A + S, A + 2 * S, stream=0)
    with pytest.raises(bh.BlackholeError):
        bh.block_norm(np.int64(0), np.int64(256), A, A + S, eps=np.float32(1e-6), stream=0)
