"""What stands between the accumulators of one block-scaled product of a transformer and the
operand of the next: the products with bias, activation and residual in their epilogue, the
gradient through that epilogue, and the norms before and after a block with its gate and residual
scale, forward and backward, over the C ABI of include/blackhole_sm100.h.

Buffers are torch tensors (checked: CUDA tensors of the current device, contiguous, of the
documented type and at least the documented size) or raw integer device pointers (taken as they
are).  Calls are asynchronous on `stream`, the current stream by default.
"""
from __future__ import annotations

import ctypes

from . import SCHEDULES, BlackholeError, _ptr, _stream, load

__all__ = ["ACTIVATIONS", "nvfp4_bf16_gemm_fused", "mxfp4_bf16_gemm_fused", "mxf8f4_bf16_gemm_fused",
           "gemm_fused_backward", "gemm_fused_backward_workspace_bytes", "NORM_KINDS", "NORM_OUTPUTS", "block_norm", "block_norm_backward",
           "block_norm_backward_workspace_bytes"]

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
NORM_KINDS = {"rms": 0, "layer": 1}
NORM_OUTPUTS = {"bf16": 0, "f32": 1, "nvfp4": 2, "mxfp4": 3, "mxfp8": 4}

_vp, _i32, _f32, _i64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_int64


class Epilogue(ctypes.Structure):
    """blackhole_sm100_epilogue"""
    _fields_ = [(n, _i32) for n in ("activation", "gated", "bias_is_bf16")] + [("beta", _f32)] + \
               [(n, _vp) for n in ("bias", "residual", "Z")]


class BlockNormArgs(ctypes.Structure):
    """blackhole_sm100_block_norm_args"""
    _fields_ = [(n, _i32) for n in ("rows", "H", "kind", "x_is_bf16", "param_is_bf16", "gate_is_bf16",
                                    "post_norm", "gate_rows", "out_format")] + \
               [(n, _f32) for n in ("eps", "scale", "global_scale")] + \
               [(n, _vp) for n in ("x", "o", "gate", "weight", "bias", "post_weight", "post_bias",
                                   "h", "out", "sf", "stats")]


class BlockNormBackwardArgs(ctypes.Structure):
    """blackhole_sm100_block_norm_backward_args"""
    _fields_ = [(n, _i32) for n in ("rows", "H", "kind", "x_is_bf16", "param_is_bf16", "gate_is_bf16",
                                    "post_norm", "gate_rows")] + [("scale", _f32)] + \
               [(n, _vp) for n in ("h", "dy", "dh", "o", "gate", "weight", "post_weight", "post_bias",
                                   "stats", "dx", "d_o", "dweight", "dbias", "dpost_weight",
                                   "dpost_bias", "dgate", "workspace")] + \
               [("workspace_bytes", _i64)]


def _torch():
    import torch
    return torch


class _Buffers:
    """Checks a call's tensors and gives their addresses.  Tensors of one `kind` (the stream, the
    parameters, the gate) share a type, BF16 or FP32."""

    def __init__(self, stream):
        self.torch = _torch()
        self.device = self.torch.cuda.current_device() if self.torch.cuda.is_available() else -1
        if stream is not None and getattr(stream, "device", None) is not None \
                and stream.device.index != self.device:
            raise ValueError(f"stream is on {stream.device}, the current device is cuda:{self.device}")
        self.kinds = {}

    def __call__(self, name, t, numel, dtype=None, kind=None):
        if t is None or type(t) is int:
            return t
        if not hasattr(t, "data_ptr"):
            raise TypeError(f"{name}: cannot take a device pointer from {type(t)!r}")
        if not t.is_cuda:
            raise ValueError(f"{name}: tensor must live on a CUDA device")
        if t.get_device() != self.device:
            raise ValueError(f"{name}: tensor is on cuda:{t.get_device()}, the current device is cuda:{self.device}")
        if not t.is_contiguous():
            raise ValueError(f"{name}: tensor must be contiguous")
        if t.numel() < numel:
            raise ValueError(f"{name}: {t.numel()} elements, {numel} are needed")
        if kind is not None:
            if self.kinds.setdefault(kind, t.dtype) != t.dtype:
                raise ValueError(f"{name}: {t.dtype}, but another tensor of its kind has {self.kinds[kind]}")
            if t.dtype not in (self.torch.bfloat16, self.torch.float32):
                raise ValueError(f"{name}: {t.dtype}, torch.bfloat16 or torch.float32 is wanted")
        elif t.dtype != dtype:
            raise ValueError(f"{name}: {t.dtype}, {dtype} is wanted")
        return t.data_ptr()

    def is_bf16(self, kind, told):
        """1 if the kind's tensors are BF16; for raw pointers what the caller says."""
        dtype = self.kinds.get(kind)
        return int(told if dtype is None else dtype == self.torch.bfloat16)


def _gate_elements(rows, H, gate_rows):
    return H * (1 if gate_rows <= 0 else -(-rows // gate_rows))


def _blocked_bytes(rows, H, vec):
    return -(-rows // 128) * -(-(H // vec) // 4) * 512


def _gemm_fused(name, M, N, K, A, SFA, B, SFB, D, alpha, bias, activation, gated, residual, beta, Z,
                bias_is_bf16, schedule, workspace, workspace_bytes, stream):
    M, N = int(M), int(N)
    b = _Buffers(stream)
    bf16 = b.torch.bfloat16
    n_out = N // 2 if gated else N
    p_d, p_res, p_z = b("D", D, M * n_out, bf16), b("residual", residual, M * n_out, bf16), b("Z", Z, M * N, bf16)
    p_bias = b("bias", bias, N, kind="bias")
    if workspace is not None and hasattr(workspace, "numel") and not workspace_bytes:
        workspace_bytes = workspace.numel() * workspace.element_size()
    epi = Epilogue(ACTIVATIONS[activation], int(bool(gated)), b.is_bf16("bias", bias_is_bf16), beta,
                   p_bias, p_res, p_z)
    rc = getattr(load(), name)(M, N, int(K), _ptr(A), _ptr(SFA), _ptr(B), _ptr(SFB), p_d, alpha,
                               ctypes.byref(epi), SCHEDULES[schedule],
                               _ptr(workspace) if workspace is not None else None,
                               int(workspace_bytes), _stream(stream))
    if rc != 0:
        raise BlackholeError(name, rc)


def nvfp4_bf16_gemm_fused(M: int, N: int, K: int, A, SFA, B, SFB, D, alpha: float = 1.0, bias=None,
                          activation: str = "none", gated: bool = False, residual=None,
                          beta: float = 1.0, Z=None, bias_is_bf16: bool = False,
                          schedule: str = "auto", workspace=None, workspace_bytes: int = 0,
                          stream=None) -> None:
    """nvfp4_bf16_gemm_ex with an epilogue fused into it:

        z = alpha * A . B^T + bias
        u = act(z), or gated: u[:, j] = act(z[:, 2j]) * z[:, 2j + 1]   (N / 2 columns)
        D = bf16(u + beta * residual)

    activation: "none", "relu", "gelu" (erf), "gelu_tanh", "silu".  gated: gate row j of the
    weights is row 2j of B, up row j row 2j + 1 (N % 16 == 0).  bias: N values, BF16 or FP32
    (bias_is_bf16 only matters for a raw pointer); residual: BF16 of D's shape, may be D itself;
    Z: BF16 M x N, receives z for gemm_fused_backward."""
    _gemm_fused("blackhole_sm100_nvfp4_bf16_gemm_fused", M, N, K, A, SFA, B, SFB, D, alpha, bias,
                activation, gated, residual, beta, Z, bias_is_bf16, schedule, workspace,
                workspace_bytes, stream)


def mxfp4_bf16_gemm_fused(M: int, N: int, K: int, A, SFA, B, SFB, D, alpha: float = 1.0, bias=None,
                          activation: str = "none", gated: bool = False, residual=None,
                          beta: float = 1.0, Z=None, bias_is_bf16: bool = False,
                          schedule: str = "auto", workspace=None, workspace_bytes: int = 0,
                          stream=None) -> None:
    """mxfp4_bf16_gemm with the epilogue of nvfp4_bf16_gemm_fused."""
    _gemm_fused("blackhole_sm100_mxfp4_bf16_gemm_fused", M, N, K, A, SFA, B, SFB, D, alpha, bias,
                activation, gated, residual, beta, Z, bias_is_bf16, schedule, workspace,
                workspace_bytes, stream)


def mxf8f4_bf16_gemm_fused(M: int, N: int, K: int, A, SFA, B, SFB, D, alpha: float = 1.0, bias=None,
                           activation: str = "none", gated: bool = False, residual=None,
                           beta: float = 1.0, Z=None, bias_is_bf16: bool = False,
                           schedule: str = "auto", workspace=None, workspace_bytes: int = 0,
                           stream=None) -> None:
    """mxf8f4_bf16_gemm with the epilogue of nvfp4_bf16_gemm_fused."""
    _gemm_fused("blackhole_sm100_mxf8f4_bf16_gemm_fused", M, N, K, A, SFA, B, SFB, D, alpha, bias,
                activation, gated, residual, beta, Z, bias_is_bf16, schedule, workspace,
                workspace_bytes, stream)


def gemm_fused_backward_workspace_bytes(M: int, N: int) -> int:
    """Workspace bytes of gemm_fused_backward's dbias (0 when none); negative for sizes it refuses."""
    return int(load().blackhole_sm100_gemm_fused_backward_workspace_bytes(int(M), int(N)))


def gemm_fused_backward(M: int, N: int, dD, Z, dZ, dbias=None, activation: str = "none",
                        gated: bool = False, workspace=None, workspace_bytes: int = 0,
                        stream=None) -> None:
    """Gradient through a fused product's epilogue, from the Z it kept: dZ = dD * act'(Z) (gated:
    of the pairs), BF16 M x N, and dbias (N FP32, overwritten; None: not wanted) its column sums.
    dD: BF16 of D's shape.  dZ may be Z, or dD when not gated.  workspace:
    gemm_fused_backward_workspace_bytes bytes, or None: allocated for this call from torch's
    caching allocator on the current stream."""
    M, N = int(M), int(N)
    b = _Buffers(stream)
    bf16 = b.torch.bfloat16
    p_d, p_z, p_dz = b("dD", dD, M * (N // 2 if gated else N), bf16), b("Z", Z, M * N, bf16), b("dZ", dZ, M * N, bf16)
    p_db = b("dbias", dbias, N, b.torch.float32)
    if workspace is None and p_db:
        need = gemm_fused_backward_workspace_bytes(M, N)
        if need > 0:
            workspace = _workspace(b, need, stream)
    if workspace is not None and type(workspace) is not int:
        workspace_bytes = workspace.numel() * workspace.element_size()
        workspace = b("workspace", workspace, 0, workspace.dtype)
    rc = load().blackhole_sm100_gemm_fused_backward(M, N, p_d, p_z, p_dz, p_db, ACTIVATIONS[activation],
                                                    int(bool(gated)), workspace, int(workspace_bytes),
                                                    _stream(stream))
    if rc != 0:
        raise BlackholeError("blackhole_sm100_gemm_fused_backward", rc)


def block_norm(rows: int, H: int, x, out=None, weight=None, bias=None, kind: str = "rms",
               eps: float = 1e-6, o=None, post_norm: bool = False, post_weight=None, post_bias=None,
               gate=None, gate_rows: int = 0, scale: float = 1.0, h=None, stats=None,
               out_format: str = "bf16", sf=None, global_scale: float = 1.0,
               x_is_bf16: bool = True, param_is_bf16: bool = False, gate_is_bf16: bool = True,
               stream=None) -> None:
    """Norms before and after a block with its gate and residual scale, one kernel:

        p = o, or norm(o) * post_weight + post_bias with post_norm
        h = x + scale * gate * p
        out = norm(h) * weight + bias

    kind "rms" or "layer".  x, h: rows x H residual stream, BF16 or FP32 (h may be x); o: BF16 or
    None (then h = x); weight, bias, post_weight, post_bias: H values, BF16 or FP32, None for 1
    and 0; gate: BF16 or FP32, row r takes gate row r // gate_rows (0: one row for all).
    out_format "bf16" or "f32", or the next product's A operand quantised from the FP32 result:
    "nvfp4" (with the caller's global_scale), "mxfp4", "mxfp8", codes in `out` (uint8) and scale
    factors in `sf` (sf_storage_bytes / mxfp4_sf_storage_bytes, padding written 0).  stats (rows x
    4 FP32) keeps what block_norm_backward needs.  The *_is_bf16 flags only matter for raw
    pointers.  rows >= 1, H % 8 == 0 (NVFP4 16, MX 32), H <= 16384.
    Raises ValueError for tensors that do not fit, BlackholeError for what the library refuses."""
    rows, H = int(rows), int(H)
    fmt = NORM_OUTPUTS[out_format]
    b = _Buffers(stream)
    bf16, f32, u8 = b.torch.bfloat16, b.torch.float32, b.torch.uint8
    n = rows * H
    out_n, out_t = ((n, bf16), (n, f32), (n // 2, u8), (n // 2, u8), (n, u8))[fmt]
    p_x, p_h = b("x", x, n, kind="x"), b("h", h, n, kind="x")
    p_o = b("o", o, n, bf16)
    p_gate = b("gate", gate, _gate_elements(rows, H, gate_rows), kind="gate")
    p_w, p_b = b("weight", weight, H, kind="param"), b("bias", bias, H, kind="param")
    p_pw, p_pb = b("post_weight", post_weight, H, kind="param"), b("post_bias", post_bias, H, kind="param")
    p_out = b("out", out, out_n, out_t)
    p_sf = b("sf", sf, _blocked_bytes(rows, H, 16 if fmt == 2 else 32), u8)
    p_st = b("stats", stats, 4 * rows, f32)
    args = BlockNormArgs(rows, H, NORM_KINDS[kind], b.is_bf16("x", x_is_bf16),
                         b.is_bf16("param", param_is_bf16), b.is_bf16("gate", gate_is_bf16),
                         int(post_norm), int(gate_rows), fmt, eps, scale, global_scale,
                         p_x, p_o, p_gate, p_w, p_b, p_pw, p_pb, p_h, p_out, p_sf, p_st)
    rc = load().blackhole_sm100_block_norm(ctypes.byref(args), _stream(stream))
    if rc != 0:
        raise BlackholeError("blackhole_sm100_block_norm", rc)


def block_norm_backward_workspace_bytes(rows: int, H: int, has_gate: bool, gate_rows: int = 0) -> int:
    """Workspace bytes of block_norm_backward for these sizes; negative for sizes it refuses."""
    return int(load().blackhole_sm100_block_norm_backward_workspace_bytes(
        int(rows), int(H), int(bool(has_gate)), int(gate_rows)))


def block_norm_backward(rows: int, H: int, h, stats, dx, dy=None, dh=None, weight=None, bias=None,
                        kind: str = "rms", eps: float = 1e-6, o=None, do=None,
                        post_norm: bool = False, post_weight=None, post_bias=None, gate=None,
                        gate_rows: int = 0, scale: float = 1.0, dweight=None, dbias=None,
                        dpost_weight=None, dpost_bias=None, dgate=None, x_is_bf16: bool = True,
                        param_is_bf16: bool = False, gate_is_bf16: bool = True, workspace=None,
                        workspace_bytes: int = 0, stream=None) -> None:
    """Gradients of block_norm.  h, stats: what it left (h: x where o was None); o, gate, weight,
    post_weight, post_bias, kind, scale, gate_rows: what it was given (bias and eps are taken for
    the same call's sake and not needed).  dy (BF16) and dh (type of x): gradients of out and h,
    None for zero; dx (type of x, may be dh) and do (BF16): written; dweight, dbias, dpost_weight,
    dpost_bias (H FP32 values) and dgate (FP32, gate's shape): overwritten where given.
    workspace: block_norm_backward_workspace_bytes bytes, or None: allocated for this call from
    torch's caching allocator on the current stream."""
    rows, H = int(rows), int(H)
    b = _Buffers(stream)
    bf16, f32 = b.torch.bfloat16, b.torch.float32
    n = rows * H
    p_h, p_st = b("h", h, n, kind="x"), b("stats", stats, 4 * rows, f32)
    p_dy, p_dh = b("dy", dy, n, bf16), b("dh", dh, n, kind="x")
    p_o, p_do, p_dx = b("o", o, n, bf16), b("do", do, n, bf16), b("dx", dx, n, kind="x")
    g_n = _gate_elements(rows, H, gate_rows)
    p_gate, p_dgate = b("gate", gate, g_n, kind="gate"), b("dgate", dgate, g_n, f32)
    p_w = b("weight", weight, H, kind="param")
    p_pw, p_pb = b("post_weight", post_weight, H, kind="param"), b("post_bias", post_bias, H, kind="param")
    p_dw, p_db = b("dweight", dweight, H, f32), b("dbias", dbias, H, f32)
    p_dpw, p_dpb = b("dpost_weight", dpost_weight, H, f32), b("dpost_bias", dpost_bias, H, f32)
    sums = p_dw or p_db or p_dpw or p_dpb or (p_dgate and gate_rows != 1)
    if workspace is None and sums:
        need = block_norm_backward_workspace_bytes(rows, H, gate is not None, gate_rows)
        if need > 0:
            workspace = _workspace(b, need, stream)
    if workspace is not None and type(workspace) is not int:
        workspace_bytes = workspace.numel() * workspace.element_size()
        workspace = b("workspace", workspace, 0, workspace.dtype)
    args = BlockNormBackwardArgs(rows, H, NORM_KINDS[kind], b.is_bf16("x", x_is_bf16),
                                 b.is_bf16("param", param_is_bf16), b.is_bf16("gate", gate_is_bf16),
                                 int(post_norm), int(gate_rows), scale, p_h, p_dy, p_dh, p_o, p_gate,
                                 p_w, p_pw, p_pb, p_st, p_dx, p_do, p_dw, p_db, p_dpw, p_dpb, p_dgate,
                                 workspace, int(workspace_bytes))
    rc = load().blackhole_sm100_block_norm_backward(ctypes.byref(args), _stream(stream))
    if rc != 0:
        raise BlackholeError("blackhole_sm100_block_norm_backward", rc)


def _workspace(b, nbytes, stream):
    """Scratch for one call on `stream`: memory the allocator hands out again only after the
    work enqueued there."""
    torch = b.torch
    if stream is None:
        return torch.empty(nbytes, dtype=torch.uint8, device=b.device)
    if isinstance(stream, int):
        stream = torch.cuda.ExternalStream(stream) if stream else torch.cuda.default_stream()
    with torch.cuda.stream(stream):
        return torch.empty(nbytes, dtype=torch.uint8, device=b.device)
