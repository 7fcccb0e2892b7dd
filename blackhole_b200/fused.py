"""What stands between the accumulators of one block-scaled product of a transformer and the
operand of the next: the products with bias, activation and residual in their epilogue, the
gradient through that epilogue, and the norms before and after a block with its gate and residual
scale, forward and backward, over the C ABI of include/blackhole_sm100.h.  Together with the quantised products they are a block's MLP:

    block_norm(.., out_format="mxfp8")            residual, norm, quantised operand
    mxf8f4_bf16_gemm_fused(.., gated=True)        gate / up projection, gated activation
    mxfp8_quantize(..)
    mxf8f4_bf16_gemm_fused(.., residual=h)        down projection, residual

Buffers are torch tensors (checked: CUDA tensors of the current device, contiguous, of the
documented type and at least the documented size) or raw integer device pointers (taken as they
are).  Calls are asynchronous on `stream`, the current stream by default.
"""
from __future__ import annotations

import struct

from . import SCHEDULES, BlackholeError, load

__all__ = ["ACTIVATIONS", "nvfp4_bf16_gemm_fused", "mxfp4_bf16_gemm_fused", "mxf8f4_bf16_gemm_fused",
           "gemm_fused_backward", "gemm_fused_backward_workspace_bytes", "NORM_KINDS", "NORM_OUTPUTS", "block_norm", "block_norm_backward",
           "block_norm_backward_workspace_bytes"]

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
NORM_KINDS = {"rms": 0, "layer": 1}
NORM_OUTPUTS = {"bf16": 0, "f32": 1, "nvfp4": 2, "mxfp4": 3, "mxfp8": 4}


# The C structs of include/blackhole_sm100.h, in their field order (native alignment); a call packs
# its arguments into bytes and passes their address.
_EPILOGUE = struct.Struct("@3if3P")             # blackhole_sm100_epilogue
_NORM = struct.Struct("@9i3f11P")               # blackhole_sm100_block_norm_args
_NORM_BACKWARD = struct.Struct("@8if17Pq")      # blackhole_sm100_block_norm_backward_args

_torch = None
_raw_stream = None


def _device():
    """torch, and the current CUDA device (-1 without one: raw pointers can still be passed)."""
    global _torch, _raw_stream
    if _torch is None:
        import torch
        _torch = torch
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    cuda = _torch.cuda
    return cuda.current_device() if cuda.is_initialized() or cuda.is_available() else -1


def _handle(stream, device):
    if stream is None:
        if device < 0:
            return 0
        if _raw_stream is not None:       # the same handle without a Stream object (1.8 us less)
            return _raw_stream(device)
        return _torch.cuda.current_stream(device).cuda_stream
    if type(stream) is int:
        return stream
    if stream.device.index != device:
        raise ValueError(f"stream is on {stream.device}, the current device is cuda:{device}")
    return stream.cuda_stream


def _at(name, t, numel, dtype, device):
    """The address of a tensor that fits (or the raw pointer, or 0 for None)."""
    if t is None:
        return 0
    if type(t) is int:
        return t
    try:
        if t.dtype is dtype and t.numel() >= numel and t.get_device() == device and t.is_contiguous() and device >= 0:
            return t.data_ptr()
    except AttributeError:
        raise TypeError(f"{name}: cannot take a device pointer from {type(t)!r}") from None
    if not t.is_cuda:
        raise ValueError(f"{name}: tensor must live on a CUDA device")
    if t.get_device() != device:
        raise ValueError(f"{name}: tensor is on {t.device}, the current device is cuda:{device}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: tensor must be contiguous")
    if t.dtype is not dtype:
        raise ValueError(f"{name}: {t.dtype}, {dtype} is wanted (tensors of one kind share a type)")
    raise ValueError(f"{name}: {t.numel()} elements, {numel} are needed")


def _operand(name, t, nbytes, device):
    """The address of a quantised operand or its scale factors: any type, at least `nbytes`."""
    if t is None:
        return 0
    if type(t) is int:
        return t
    try:
        size = t.numel() * t.element_size()
    except AttributeError:
        raise TypeError(f"{name}: cannot take a device pointer from {type(t)!r}") from None
    if size < nbytes:
        raise ValueError(f"{name}: {size} bytes, {nbytes} are needed")
    return _at(name, t, 0, t.dtype, device)


def _kind(told_bf16, *tensors):
    """The type of a call's tensors of one kind (the stream, the parameters, the gate): that of the
    first one given, BF16 or FP32; for raw pointers what the caller says."""
    for t in tensors:
        dtype = getattr(t, "dtype", None)
        if dtype is not None:
            if dtype is not _torch.bfloat16 and dtype is not _torch.float32:
                raise ValueError(f"{dtype}: torch.bfloat16 or torch.float32 is wanted")
            return dtype
    return _torch.bfloat16 if told_bf16 else _torch.float32


def _gate_elements(rows, H, gate_rows):
    return H * (1 if gate_rows <= 0 else -(-rows // gate_rows))


def _blocked_bytes(rows, H, vec):
    return -(-rows // 128) * -(-(H // vec) // 4) * 512


def _gemm_fused(fmt, M, N, K, A, SFA, B, SFB, D, alpha, bias, activation, gated, residual, beta, Z,
                bias_is_bf16, schedule, workspace, workspace_bytes, stream):
    M, N, K, dev = int(M), int(N), int(K), _device()
    handle, bf16 = _handle(stream, dev), _torch.bfloat16
    n = M * (N // 2 if gated else N)
    t_bias = _kind(bias_is_bf16, bias)
    epi = _EPILOGUE.pack(ACTIVATIONS[activation], 1 if gated else 0, t_bias is bf16, beta,
                         _at("bias", bias, N, t_bias, dev), _at("residual", residual, n, bf16, dev),
                         _at("Z", Z, M * N, bf16, dev))
    if hasattr(workspace, "numel"):
        workspace_bytes = workspace.numel() * workspace.element_size()
    vec = 16 if fmt == "nvfp4" else 32
    name = f"blackhole_sm100_{fmt}_bf16_gemm_fused"
    rc = getattr(load(), name)(
        M, N, K, _operand("A", A, M * K if fmt == "mxf8f4" else M * K // 2, dev),
        _operand("SFA", SFA, _blocked_bytes(M, K, vec), dev), _operand("B", B, N * K // 2, dev),
        _operand("SFB", SFB, _blocked_bytes(N, K, vec), dev), _at("D", D, n, bf16, dev), float(alpha), epi,
        SCHEDULES[schedule], _operand("workspace", workspace, 0, dev), workspace_bytes, handle)
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
    _gemm_fused("nvfp4", M, N, K, A, SFA, B, SFB, D, alpha, bias,
                activation, gated, residual, beta, Z, bias_is_bf16, schedule, workspace,
                workspace_bytes, stream)


def mxfp4_bf16_gemm_fused(M: int, N: int, K: int, A, SFA, B, SFB, D, alpha: float = 1.0, bias=None,
                          activation: str = "none", gated: bool = False, residual=None,
                          beta: float = 1.0, Z=None, bias_is_bf16: bool = False,
                          schedule: str = "auto", workspace=None, workspace_bytes: int = 0,
                          stream=None) -> None:
    """mxfp4_bf16_gemm with the epilogue of nvfp4_bf16_gemm_fused."""
    _gemm_fused("mxfp4", M, N, K, A, SFA, B, SFB, D, alpha, bias,
                activation, gated, residual, beta, Z, bias_is_bf16, schedule, workspace,
                workspace_bytes, stream)


def mxf8f4_bf16_gemm_fused(M: int, N: int, K: int, A, SFA, B, SFB, D, alpha: float = 1.0, bias=None,
                           activation: str = "none", gated: bool = False, residual=None,
                           beta: float = 1.0, Z=None, bias_is_bf16: bool = False,
                           schedule: str = "auto", workspace=None, workspace_bytes: int = 0,
                           stream=None) -> None:
    """mxf8f4_bf16_gemm with the epilogue of nvfp4_bf16_gemm_fused."""
    _gemm_fused("mxf8f4", M, N, K, A, SFA, B, SFB, D, alpha, bias,
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
    M, N, dev = int(M), int(N), _device()
    handle, bf16 = _handle(stream, dev), _torch.bfloat16
    p_db = _at("dbias", dbias, N, _torch.float32, dev)
    need = gemm_fused_backward_workspace_bytes(M, N) if p_db and workspace is None else 0
    p_ws, workspace_bytes, workspace = _scratch(workspace, workspace_bytes, need, stream, dev)
    rc = load().blackhole_sm100_gemm_fused_backward(
        M, N, _at("dD", dD, M * (N // 2 if gated else N), bf16, dev), _at("Z", Z, M * N, bf16, dev),
        _at("dZ", dZ, M * N, bf16, dev), p_db, ACTIVATIONS[activation], 1 if gated else 0, p_ws,
        workspace_bytes, handle)
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
    dev = _device()
    handle, fmt, n = _handle(stream, dev), NORM_OUTPUTS[out_format], rows * H
    bf16, f32, u8 = _torch.bfloat16, _torch.float32, _torch.uint8
    out_n, out_t = ((n, bf16), (n, f32), (n // 2, u8), (n // 2, u8), (n, u8))[fmt]
    tx, tp, tg = (_kind(x_is_bf16, x), _kind(param_is_bf16, weight, bias, post_weight, post_bias),
                  _kind(gate_is_bf16, gate))
    args = _NORM.pack(
        rows, H, NORM_KINDS[kind], tx is bf16, tp is bf16, tg is bf16, bool(post_norm), gate_rows, fmt,
        eps, scale, global_scale,
        _at("x", x, n, tx, dev), _at("o", o, n, bf16, dev),
        _at("gate", gate, _gate_elements(rows, H, gate_rows), tg, dev),
        _at("weight", weight, H, tp, dev), _at("bias", bias, H, tp, dev),
        _at("post_weight", post_weight, H, tp, dev), _at("post_bias", post_bias, H, tp, dev),
        _at("h", h, n, tx, dev), _at("out", out, out_n, out_t, dev),
        _at("sf", sf, _blocked_bytes(rows, H, 16 if fmt == 2 else 32), u8, dev),
        _at("stats", stats, 4 * rows, f32, dev))
    rc = load().blackhole_sm100_block_norm(args, handle)
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
    dev = _device()
    handle, n, g_n = _handle(stream, dev), rows * H, _gate_elements(rows, H, gate_rows)
    bf16, f32 = _torch.bfloat16, _torch.float32
    tx, tp, tg = (_kind(x_is_bf16, h), _kind(param_is_bf16, weight, post_weight, post_bias),
                  _kind(gate_is_bf16, gate))
    sums = [_at("dweight", dweight, H, f32, dev), _at("dbias", dbias, H, f32, dev),
            _at("dpost_weight", dpost_weight, H, f32, dev), _at("dpost_bias", dpost_bias, H, f32, dev),
            _at("dgate", dgate, g_n, f32, dev)]
    need = 0
    if workspace is None and (any(sums[:4]) or (sums[4] and gate_rows != 1)):
        need = block_norm_backward_workspace_bytes(rows, H, gate is not None, gate_rows)
    p_ws, workspace_bytes, workspace = _scratch(workspace, workspace_bytes, need, stream, dev)
    args = _NORM_BACKWARD.pack(
        rows, H, NORM_KINDS[kind], tx is bf16, tp is bf16, tg is bf16, bool(post_norm), gate_rows, scale,
        _at("h", h, n, tx, dev), _at("dy", dy, n, bf16, dev), _at("dh", dh, n, tx, dev),
        _at("o", o, n, bf16, dev), _at("gate", gate, g_n, tg, dev), _at("weight", weight, H, tp, dev),
        _at("post_weight", post_weight, H, tp, dev), _at("post_bias", post_bias, H, tp, dev),
        _at("stats", stats, 4 * rows, f32, dev), _at("dx", dx, n, tx, dev), _at("do", do, n, bf16, dev),
        *sums, p_ws, workspace_bytes)
    rc = load().blackhole_sm100_block_norm_backward(args, handle)
    if rc != 0:
        raise BlackholeError("blackhole_sm100_block_norm_backward", rc)


def _scratch(workspace, workspace_bytes, need, stream, device):
    """(address, bytes, owner) of a call's workspace: the caller's, or `need` bytes of torch's
    caching allocator on `stream`, which hands them out again only after the work enqueued there."""
    if workspace is None:
        if need <= 0 or device < 0:
            return 0, 0, None
        if stream is None:
            workspace = _torch.empty(need, dtype=_torch.uint8, device=device)
        else:
            if type(stream) is int:
                stream = _torch.cuda.ExternalStream(stream) if stream else _torch.cuda.default_stream()
            with _torch.cuda.stream(stream):
                workspace = _torch.empty(need, dtype=_torch.uint8, device=device)
        return workspace.data_ptr(), need, workspace
    if type(workspace) is int:
        return workspace, workspace_bytes, workspace
    return (_at("workspace", workspace, 0, workspace.dtype, device),
            workspace.numel() * workspace.element_size(), workspace)
