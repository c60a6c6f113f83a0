"""ctypes binding of `lib/libmamba3_amd.so` (C-ABI declared in include/mamba3_amd.h).

PyTorch supplies device memory and the current HIP stream; every compute call goes
through the native library. There is no CPU or eager fallback: a CPU tensor or a
missing library raises.
"""

from __future__ import annotations

import ctypes
import functools
import threading
from array import array
from pathlib import Path

import torch

LIB_PATH = Path(__file__).resolve().parent / "lib" / "libmamba3_amd.so"

M3_DTYPE_F32 = 0
M3_DTYPE_BF16 = 1

_DTYPE_CODE = {torch.float32: M3_DTYPE_F32, torch.bfloat16: M3_DTYPE_BF16}

# Exported symbols, kept in step with include/mamba3_amd.h.
EXPORTED_SYMBOLS = (
    "m3_status_string",
    "m3_version",
    "m3_scan_fwd",
    "m3_scan_bwd_workspace_size",
    "m3_scan_bwd",
    "m3_prefill_workspace_size",
    "m3_prefill_fwd",
    "m3_step_fwd",
    "m3_chunked_ssd_fwd",
    "m3_chunked_ssd_fwd_workspace_size",
    "m3_chunked_ssd_bwd_workspace_size",
    "m3_chunked_ssd_bwd",
    "m3_layer_bwd_workspace_size",
    "m3_layer_bwd",
    "m3_prefill_fwd_noalloc",
    "m3_rmsnorm_fwd",
    "m3_rmsnorm_bwd_workspace_size",
    "m3_rmsnorm_bwd",
    "m3_small_linear",
    "m3_small_swiglu",
    "m3_silu_mul",
    "m3_step_bwd_workspace_size",
    "m3_step_bwd",
    "m3_prefill_kernel_name",
    "m3_swiglu_mlp_saved_size",
    "m3_swiglu_mlp_fwd_workspace_size",
    "m3_swiglu_mlp_fwd",
    "m3_swiglu_mlp_bwd_workspace_size",
    "m3_swiglu_mlp_bwd",
    "m3_linear_xent_fwd_workspace_size",
    "m3_linear_xent_fwd",
    "m3_linear_xent_bwd_workspace_size",
    "m3_linear_xent_bwd",
    "m3_clip_grad_norm_workspace_size",
    "m3_clip_grad_norm",
    "m3_mx_quantize",
    "m3_mx_dequantize",
    "m3_add_rmsnorm_fwd",
    "m3_add_rmsnorm_mx",
    "m3_add_rmsnorm_bwd_workspace_size",
    "m3_add_rmsnorm_bwd",
    "m3_mx_linear",
    "m3_mx_linear_exact",
    "m3_mx_linear_exact_workspace_size",
    "m3_mx_linear_takes_tensor",
    "m3_mx_linear_tensor",
    "m3_sample_tokens",
)

M3_ERR_UNSUPPORTED = 3
M3_ERR_WORKSPACE = 4
M3_ERR_SCRATCH_LIMIT = 8
M3_ERR_OVERLAP = 9
NOALLOC_SCRATCH_BYTES = 64 << 20


class NativeError(RuntimeError):
    """A native entry point returned a non-zero m3_status (in `status`)."""

    status = None


class LayerDesc(ctypes.Structure):
    _fields_ = [
        ("batch", ctypes.c_int32),
        ("seqlen", ctypes.c_int32),
        ("nheads", ctypes.c_int32),
        ("headdim", ctypes.c_int32),
        ("d_state", ctypes.c_int32),
        ("mimo_rank", ctypes.c_int32),
        ("ngroups", ctypes.c_int32),
        ("use_trapezoidal", ctypes.c_int32),
        ("use_complex", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("proj_row_stride", ctypes.c_int64),
        ("rms_eps", ctypes.c_float),
        ("flags", ctypes.c_int32),
    ]


M3_FLAG_NO_F16_OPERANDS = 1
M3_FLAG_FOR_BACKWARD = 2


class LayerParams(ctypes.Structure):
    _fields_ = [(name, ctypes.c_void_p) for name in (
        "A_log", "D", "dt_bias", "B_norm_w", "C_norm_w", "B_bias", "C_bias",
        "mimo_x", "mimo_z", "mimo_down")]


class LayerParamGrads(ctypes.Structure):
    _fields_ = LayerParams._fields_ + [("dt_scale", ctypes.c_void_p)]


_lib = None
_lib_lock = threading.Lock()

_vp = ctypes.c_void_p
_i32 = ctypes.c_int32
_i64 = ctypes.c_int64


def _declare(lib: ctypes.CDLL) -> None:
    lib.m3_status_string.restype = ctypes.c_char_p
    lib.m3_status_string.argtypes = [ctypes.c_int]
    lib.m3_version.restype = ctypes.c_int
    lib.m3_version.argtypes = []
    lib.m3_scan_fwd.restype = ctypes.c_int
    lib.m3_scan_fwd.argtypes = [_vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _vp]
    lib.m3_scan_bwd_workspace_size.restype = ctypes.c_int
    lib.m3_scan_bwd_workspace_size.argtypes = [_i64, _i64, _i64, _i64, ctypes.POINTER(ctypes.c_size_t)]
    lib.m3_scan_bwd.restype = ctypes.c_int
    lib.m3_scan_bwd.argtypes = [_vp, _vp, _vp, _vp, _vp, _vp, _vp, ctypes.c_size_t,
                                _i64, _i64, _i64, _i64, _vp]
    lib.m3_prefill_kernel_name.restype = ctypes.c_char_p
    lib.m3_prefill_kernel_name.argtypes = [ctypes.POINTER(LayerDesc), _vp, _vp, _vp, _vp]
    lib.m3_prefill_workspace_size.restype = ctypes.c_int
    lib.m3_prefill_workspace_size.argtypes = [ctypes.POINTER(LayerDesc),
                                              ctypes.POINTER(ctypes.c_size_t)]
    lib.m3_prefill_fwd.restype = ctypes.c_int
    lib.m3_prefill_fwd.argtypes = [ctypes.POINTER(LayerDesc), ctypes.POINTER(LayerParams),
                                   _vp, _vp, _vp, _vp, _vp, _vp, _vp, ctypes.c_size_t, _vp]
    lib.m3_prefill_fwd_noalloc.restype = ctypes.c_int
    lib.m3_prefill_fwd_noalloc.argtypes = [ctypes.POINTER(LayerDesc), ctypes.POINTER(LayerParams),
                                           _vp, _vp, _vp, _vp, _vp, _vp, _vp]
    lib.m3_rmsnorm_fwd.restype = ctypes.c_int
    lib.m3_rmsnorm_fwd.argtypes = [_vp, ctypes.c_int, _vp, ctypes.c_int, _vp, ctypes.c_int, _vp,
                                   _i64, _i32, ctypes.c_float, _vp]
    lib.m3_rmsnorm_bwd_workspace_size.restype = ctypes.c_int
    lib.m3_rmsnorm_bwd_workspace_size.argtypes = [_i64, _i32, ctypes.POINTER(ctypes.c_size_t)]
    lib.m3_rmsnorm_bwd.restype = ctypes.c_int
    lib.m3_rmsnorm_bwd.argtypes = [_vp, ctypes.c_int, _vp, ctypes.c_int, _vp, _vp, ctypes.c_int,
                                   _vp, _vp, _vp, ctypes.c_size_t, _i64, _i32, _vp]
    lib.m3_small_linear.restype = ctypes.c_int
    lib.m3_small_linear.argtypes = [_vp, _vp, ctypes.c_float, _vp, _vp, ctypes.c_float, _vp,
                                    _i32, _i32, _i32, _vp]
    lib.m3_silu_mul.restype = ctypes.c_int
    lib.m3_silu_mul.argtypes = [_vp, _i64, _i32, _i64, _vp, _vp]
    lib.m3_small_swiglu.restype = ctypes.c_int
    lib.m3_small_swiglu.argtypes = [_vp, _vp, ctypes.c_float, _vp, _vp, _vp, _i32, _i32, _i32, _vp]
    lib.m3_step_fwd.restype = ctypes.c_int
    lib.m3_step_fwd.argtypes = [ctypes.POINTER(LayerDesc), ctypes.POINTER(LayerParams),
                                _vp, _vp, _vp, _vp, _vp, ctypes.c_int, _vp, _vp, _vp, _vp, _vp]
    lib.m3_chunked_ssd_fwd.restype = ctypes.c_int
    lib.m3_chunked_ssd_fwd.argtypes = [_i32, _i32, _i32, _i32, _i32, _i32, _i32,
                                       _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp,
                                       _vp, _vp, _vp, _vp, ctypes.c_size_t, _vp]
    lib.m3_chunked_ssd_fwd_workspace_size.restype = ctypes.c_int
    lib.m3_chunked_ssd_fwd_workspace_size.argtypes = [_i32] * 8 + [ctypes.POINTER(ctypes.c_size_t)]
    lib.m3_layer_bwd_workspace_size.restype = ctypes.c_int
    lib.m3_layer_bwd_workspace_size.argtypes = [ctypes.POINTER(LayerDesc), ctypes.POINTER(ctypes.c_size_t)]
    lib.m3_layer_bwd.restype = ctypes.c_int
    lib.m3_layer_bwd.argtypes = ([ctypes.POINTER(LayerDesc), ctypes.POINTER(LayerParams)]
                                 + [_vp] * 3 + [ctypes.c_size_t] + [_vp] * 5
                                 + [ctypes.POINTER(LayerParamGrads), _vp, ctypes.c_size_t, _vp])
    lib.m3_step_bwd_workspace_size.restype = ctypes.c_int
    lib.m3_step_bwd_workspace_size.argtypes = [ctypes.POINTER(LayerDesc), ctypes.POINTER(ctypes.c_size_t)]
    lib.m3_step_bwd.restype = ctypes.c_int
    lib.m3_step_bwd.argtypes = ([ctypes.POINTER(LayerDesc), ctypes.POINTER(LayerParams)]
                                + [_vp] * 13
                                + [ctypes.POINTER(LayerParamGrads), _vp, ctypes.c_size_t, _vp])
    lib.m3_chunked_ssd_bwd_workspace_size.restype = ctypes.c_int
    lib.m3_chunked_ssd_bwd_workspace_size.argtypes = [_i32] * 7 + [ctypes.POINTER(ctypes.c_size_t)]
    lib.m3_chunked_ssd_bwd.restype = ctypes.c_int
    lib.m3_chunked_ssd_bwd.argtypes = [_i32] * 6 + [_vp] * 23 + [ctypes.c_size_t, _vp]
    size_p, f32 = ctypes.POINTER(ctypes.c_size_t), ctypes.c_float
    dims = [_i64, _i32, _i32, _i32]  # rows, d_model, d_ff or vocab, dtype
    for name, args in (
            ("m3_swiglu_mlp_saved_size", [*dims, size_p]),
            ("m3_swiglu_mlp_fwd_workspace_size", [*dims, _i32, size_p]),
            ("m3_swiglu_mlp_fwd", [*dims] + [_vp] * 5 + [f32] + [_vp] * 3 + [ctypes.c_size_t, _vp]),
            ("m3_swiglu_mlp_bwd_workspace_size", [*dims, size_p]),
            ("m3_swiglu_mlp_bwd", [*dims] + [_vp] * 4 + [f32] + [_vp] * 7 + [ctypes.c_size_t, _vp]),
            ("m3_linear_xent_fwd_workspace_size", [*dims, size_p]),
            ("m3_linear_xent_fwd", [*dims, _i32] + [_vp] * 3 + [_i64] + [_vp] * 4 + [ctypes.c_size_t, _vp]),
            ("m3_linear_xent_bwd_workspace_size", [*dims, _i32, _i32, size_p]),
            ("m3_linear_xent_bwd", [*dims, _i32] + [_vp] * 3 + [_i64] + [_vp] * 6 + [ctypes.c_size_t, _vp]),
            ("m3_clip_grad_norm_workspace_size", [_i32, _vp, _vp, size_p]),
            ("m3_clip_grad_norm", [_i32, _vp, _vp, _vp, _i32, _i32, f32] + [_vp] * 2 + [ctypes.c_size_t, _vp]),
            ("m3_mx_quantize", [_i64] + [_i32] * 4 + [_vp] * 4),
            ("m3_mx_dequantize", [_i64] + [_i32] * 3 + [_vp] * 4),
            ("m3_add_rmsnorm_fwd", [_i64, _i32, _i32] + [_vp] * 3 + [f32, f32] + [_vp] * 4),
            ("m3_add_rmsnorm_mx", [_i64, _i32, _i32] + [_vp] * 3 + [f32, f32, _vp, _i32] + [_vp] * 3),
            ("m3_add_rmsnorm_bwd_workspace_size", [_i64, _i32, size_p]),
            ("m3_add_rmsnorm_bwd", [_i64, _i32, _i32] + [_vp] * 5 + [f32] + [_vp] * 4 + [ctypes.c_size_t, _vp]),
            ("m3_mx_linear", [_i64] + [_i32] * 4 + [_vp] * 5 + [f32] + [_vp] * 2),
            ("m3_mx_linear_exact", [_i64] + [_i32] * 3 + [_vp] * 5 + [f32] + [_vp] * 2 + [ctypes.c_size_t, _vp]),
            ("m3_mx_linear_exact_workspace_size", [_i64] + [_i32] * 2 + [ctypes.POINTER(ctypes.c_size_t)]),
            ("m3_mx_linear_takes_tensor", [_i64] + [_i32] * 5),
            ("m3_mx_linear_tensor", [_i64] + [_i32] * 5 + [_vp] * 2 + [f32] + [_vp] * 3 + [f32] + [_vp] * 2),
            ("m3_sample_tokens", [_i64, _i32, _i32, _vp, _vp, _vp, ctypes.c_double, _vp, _i64, _vp, ctypes.c_double, _vp,
                                  ctypes.c_double, _vp, _vp, _vp])):
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = ctypes.c_int, args


def lib() -> ctypes.CDLL:
    """Load the native library (once). Raises if it has not been built."""
    global _lib
    if _lib is None:
        with _lib_lock:
            if _lib is None:
                if not LIB_PATH.exists():
                    raise RuntimeError(
                        f"mamba3_amd native library not found at {LIB_PATH}; "
                        "build it with `python -m mamba3_amd.build`")
                handle = ctypes.CDLL(str(LIB_PATH))
                _declare(handle)
                _lib = handle
    return _lib


def check(status: int, what: str) -> None:
    if status != 0:
        msg = lib().m3_status_string(status).decode()
        err = NativeError(f"{what}: {msg} (m3_status {status})")
        err.status = status
        raise err


def dtype_code(dtype: torch.dtype) -> int:
    try:
        return _DTYPE_CODE[dtype]
    except KeyError:
        raise TypeError(f"mamba3_amd kernels support float32 and bfloat16, got {dtype}") from None


def require_gpu(*tensors: torch.Tensor) -> None:
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise RuntimeError(
                "mamba3_amd runs its SSD path only as HIP kernels on an AMD GPU; "
                f"got a tensor on {t.device}. Move the module and inputs to the GPU.")


def ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


# The current stream's handle by device index, without the Stream object that
# torch.cuda.current_stream builds (4 us a call; a decode step makes three).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def stream_of(t: torch.Tensor) -> int:
    if _raw_stream is None:
        return torch.cuda.current_stream(t.device).cuda_stream
    return _raw_stream(t.get_device())


def scan_fwd(decay: torch.Tensor, h_chunk: torch.Tensor, h_init: torch.Tensor | None,
             out: torch.Tensor) -> None:
    B, K, H, PN = h_chunk.shape
    check(lib().m3_scan_fwd(ptr(decay), ptr(h_chunk), ptr(h_init), ptr(out), B, K, H, PN,
                            stream_of(h_chunk)), "m3_scan_fwd")


def scan_bwd(decay: torch.Tensor, h_states: torch.Tensor, grad: torch.Tensor,
             d_decay: torch.Tensor, d_chunk: torch.Tensor, d_h_init: torch.Tensor | None) -> None:
    """m3_scan_bwd on contiguous fp32 tensors (B,K,H) / (B,K,H,PN) / (B,H,PN)."""
    B, K, H, PN = h_states.shape
    n = ctypes.c_size_t(0)
    check(lib().m3_scan_bwd_workspace_size(B, K, H, PN, ctypes.byref(n)), "m3_scan_bwd_workspace_size")
    ws = torch.empty(max(n.value, 1), dtype=torch.uint8, device=h_states.device)
    check(lib().m3_scan_bwd(ptr(decay), ptr(h_states), ptr(grad), ptr(d_decay), ptr(d_chunk),
                            ptr(d_h_init), ptr(ws), n.value, B, K, H, PN, stream_of(h_states)),
          "m3_scan_bwd")


def prefill_workspace_bytes(desc: LayerDesc) -> int:
    n = ctypes.c_size_t(0)
    check(lib().m3_prefill_workspace_size(ctypes.byref(desc), ctypes.byref(n)),
          "m3_prefill_workspace_size")
    return n.value


def prefill_kernel_name(desc: LayerDesc, proj=None, y_out=None, h_final=None, prev_bx=None) -> str:
    """Name of the prefill kernel m3_prefill_fwd runs for these arguments."""
    name = lib().m3_prefill_kernel_name(ctypes.byref(desc), ptr(proj), ptr(y_out), ptr(h_final),
                                        ptr(prev_bx))
    if name is None:
        raise NativeError("m3_prefill_kernel_name: invalid layer descriptor")
    return name.decode()


def prefill_fwd(desc: LayerDesc, params: LayerParams, proj, dt_scale, y_out, h_final, angle,
                prev_bx, workspace, workspace_bytes: int) -> None:
    st = lib().m3_prefill_fwd(ctypes.byref(desc), ctypes.byref(params), proj.data_ptr(),
                              ptr(dt_scale), y_out.data_ptr(), ptr(h_final), ptr(angle),
                              ptr(prev_bx), ptr(workspace), workspace_bytes, stream_of(proj))
    if st:
        check(st, "m3_prefill_fwd")


def prefill_fwd_noalloc(desc: LayerDesc, params: LayerParams, proj, dt_scale, y_out, h_final,
                        angle, prev_bx) -> None:
    """m3_prefill_fwd_noalloc: m3_prefill_fwd on the library's static per-device scratch."""
    check(lib().m3_prefill_fwd_noalloc(ctypes.byref(desc), ctypes.byref(params), ptr(proj),
                                       ptr(dt_scale), ptr(y_out), ptr(h_final), ptr(angle),
                                       ptr(prev_bx), stream_of(proj)), "m3_prefill_fwd_noalloc")


def step_fwd(desc: LayerDesc, params: LayerParams, proj, dt_scale, h_in, prev_in, angle_in,
             y_out, h_out, prev_out, angle_out) -> None:
    st = lib().m3_step_fwd(ctypes.byref(desc), ctypes.byref(params), proj.data_ptr(),
                           ptr(dt_scale), h_in.data_ptr(), prev_in.data_ptr(), angle_in.data_ptr(),
                           dtype_code(angle_in.dtype), y_out.data_ptr(), h_out.data_ptr(),
                           prev_out.data_ptr(), angle_out.data_ptr(), stream_of(proj))
    if st:
        check(st, "m3_step_fwd")


def chunked_fwd_mfma_applies(B, T, H, P, N, R, has_beta: bool) -> bool:
    """True when m3_chunked_ssd_fwd runs fp32 inputs of this shape on its fp32-MFMA path."""
    n = ctypes.c_size_t(0)
    check(lib().m3_chunked_ssd_fwd_workspace_size(B, T, H, P, N, R, 0, int(has_beta),
                                                  ctypes.byref(n)),
          "m3_chunked_ssd_fwd_workspace_size")
    return n.value > 0


def chunked_fwd(B, T, H, P, N, R, dtype, x_g, x_b, B_g, B_b, C, dt, A, D, x_raw, h_init, y,
                h_final, state_ws, use_workspace: bool = True) -> None:
    """m3_chunked_ssd_fwd; allocates the workspace of the fp32-MFMA path when it applies
    (use_workspace=False runs the generic kernel)."""
    n = ctypes.c_size_t(0)
    check(lib().m3_chunked_ssd_fwd_workspace_size(B, T, H, P, N, R, dtype_code(dtype),
                                                  int(x_b is not None), ctypes.byref(n)),
          "m3_chunked_ssd_fwd_workspace_size")
    if not use_workspace:
        n.value = 0
    ws = torch.empty(n.value, dtype=torch.uint8, device=x_g.device) if n.value else None
    check(lib().m3_chunked_ssd_fwd(B, T, H, P, N, R, dtype_code(dtype), ptr(x_g), ptr(x_b),
                                   ptr(B_g), ptr(B_b), ptr(C), ptr(dt), ptr(A), ptr(D),
                                   ptr(x_raw), ptr(h_init), ptr(y), ptr(h_final),
                                   ptr(state_ws), ptr(ws), n.value, stream_of(x_g)),
          "m3_chunked_ssd_fwd")


def chunked_bwd_workspace_bytes(B, T, H, P, N, R, has_beta: bool) -> int:
    n = ctypes.c_size_t(0)
    check(lib().m3_chunked_ssd_bwd_workspace_size(B, T, H, P, N, R, int(has_beta), ctypes.byref(n)),
          "m3_chunked_ssd_bwd_workspace_size")
    return n.value


def chunked_bwd(B, T, H, P, N, R, x_g, x_b, B_g, B_b, C, dt, A, D, x_raw, h_init, dy, dh_final,
                dx_g, dx_b, dB_g, dB_b, dC, ddt, dA, dD, dx_raw, dh_init) -> None:
    """m3_chunked_ssd_bwd on contiguous fp32 tensors; allocates the workspace."""
    n = chunked_bwd_workspace_bytes(B, T, H, P, N, R, x_b is not None)
    ws = torch.empty(max(n, 1), dtype=torch.uint8, device=x_g.device)
    check(lib().m3_chunked_ssd_bwd(B, T, H, P, N, R, ptr(x_g), ptr(x_b), ptr(B_g), ptr(B_b),
                                   ptr(C), ptr(dt), ptr(A), ptr(D), ptr(x_raw), ptr(h_init),
                                   ptr(dy), ptr(dh_final), ptr(dx_g), ptr(dx_b), ptr(dB_g),
                                   ptr(dB_b), ptr(dC), ptr(ddt), ptr(dA), ptr(dD), ptr(dx_raw),
                                   ptr(dh_init), ptr(ws), n, stream_of(x_g)),
          "m3_chunked_ssd_bwd")


def layer_bwd_supported(desc: LayerDesc) -> bool:
    """True when m3_layer_bwd covers this (fp32) layer shape."""
    n = ctypes.c_size_t(0)
    st = lib().m3_layer_bwd_workspace_size(ctypes.byref(desc), ctypes.byref(n))
    return st == 0 and n.value > 0


def layer_bwd_workspace_bytes(desc: LayerDesc) -> int:
    n = ctypes.c_size_t(0)
    check(lib().m3_layer_bwd_workspace_size(ctypes.byref(desc), ctypes.byref(n)),
          "m3_layer_bwd_workspace_size")
    return n.value


def layer_bwd(desc: LayerDesc, params: LayerParams, proj, dt_scale, fwd_ws, g_out, g_h, g_angle,
              g_prev, g_proj, grads: LayerParamGrads) -> None:
    """m3_layer_bwd; allocates its workspace."""
    n = layer_bwd_workspace_bytes(desc)
    ws = torch.empty(n, dtype=torch.uint8, device=proj.device)
    check(lib().m3_layer_bwd(ctypes.byref(desc), ctypes.byref(params), ptr(proj), ptr(dt_scale),
                             ptr(fwd_ws), fwd_ws.numel(), ptr(g_out), ptr(g_h), ptr(g_angle),
                             ptr(g_prev), ptr(g_proj), ctypes.byref(grads), ptr(ws), n,
                             stream_of(proj)),
          "m3_layer_bwd")


def step_bwd_supported(desc: LayerDesc) -> bool:
    """True when m3_step_bwd covers this (fp32) layer shape."""
    n = ctypes.c_size_t(0)
    st = lib().m3_step_bwd_workspace_size(ctypes.byref(desc), ctypes.byref(n))
    return st == 0 and n.value > 0


def step_bwd(desc: LayerDesc, params: LayerParams, proj, dt_scale, h_in, prev_in, angle_in, g_y,
             g_h, g_prev, g_angle, g_proj, g_h_in, g_prev_in, g_angle_in,
             grads: LayerParamGrads) -> None:
    """m3_step_bwd; allocates its workspace."""
    n = ctypes.c_size_t(0)
    check(lib().m3_step_bwd_workspace_size(ctypes.byref(desc), ctypes.byref(n)),
          "m3_step_bwd_workspace_size")
    ws = torch.empty(n.value, dtype=torch.uint8, device=proj.device)
    check(lib().m3_step_bwd(ctypes.byref(desc), ctypes.byref(params), ptr(proj), ptr(dt_scale),
                            ptr(h_in), ptr(prev_in), ptr(angle_in), ptr(g_y), ptr(g_h),
                            ptr(g_prev), ptr(g_angle), ptr(g_proj), ptr(g_h_in), ptr(g_prev_in),
                            ptr(g_angle_in), ctypes.byref(grads), ptr(ws), n.value,
                            stream_of(proj)),
          "m3_step_bwd")


def rmsnorm_fwd(x, weight, y, rstd, eps: float) -> None:
    """m3_rmsnorm_fwd on contiguous x (rows, d)."""
    rows, d = x.shape
    st = lib().m3_rmsnorm_fwd(x.data_ptr(), dtype_code(x.dtype), weight.data_ptr(),
                              dtype_code(weight.dtype), y.data_ptr(), dtype_code(y.dtype),
                              ptr(rstd), rows, d, eps, stream_of(x))
    if st:
        check(st, "m3_rmsnorm_fwd")


SMALL_PROJ_MAX_ROWS = 8


def small_proj_ok(m: int, k: int, norm: bool = False) -> bool:
    """The shapes m3_small_linear / m3_small_swiglu take: m <= 8 rows, k a multiple of 64
    whose staged rows (m rounded up to 1, 2, 4 or 8) and, with a norm, the norm weight fit
    64 KB of LDS."""
    mm = 1 if m <= 1 else 2 if m <= 2 else 4 if m <= 4 else 8
    need = (mm * k + 8 + (k if norm else 0)) * 2
    return 1 <= m <= SMALL_PROJ_MAX_ROWS and k >= 64 and k % 64 == 0 and need <= 65536


def small_linear(x, norm_w, eps, weight, residual, scale, out) -> None:
    """m3_small_linear on contiguous bf16 x (m, k), weight (n, k), out (m, n)."""
    m, k = x.shape
    st = lib().m3_small_linear(x.data_ptr(), ptr(norm_w), eps, weight.data_ptr(), ptr(residual),
                               scale, out.data_ptr(), m, weight.shape[0], k, stream_of(x))
    if st:
        check(st, "m3_small_linear")


def small_swiglu(x, norm_w, eps, w_gate, w_up, out) -> None:
    """m3_small_swiglu on contiguous bf16 x (m, k), weights (n, k), out (m, n)."""
    m, k = x.shape
    st = lib().m3_small_swiglu(x.data_ptr(), ptr(norm_w), eps, w_gate.data_ptr(), w_up.data_ptr(),
                               out.data_ptr(), m, w_gate.shape[0], k, stream_of(x))
    if st:
        check(st, "m3_small_swiglu")


def silu_mul(gate_up, d_ff, out) -> None:
    """m3_silu_mul on bf16 gate_up (rows, >= 2 d_ff) with unit column stride."""
    check(lib().m3_silu_mul(ptr(gate_up), gate_up.shape[0], d_ff, gate_up.stride(0), ptr(out),
                            stream_of(gate_up)), "m3_silu_mul")


def rmsnorm_bwd(x, weight, rstd, grad, dx, dweight) -> None:
    """m3_rmsnorm_bwd on contiguous (rows, d) tensors; allocates the workspace."""
    rows, d = x.shape
    n = ctypes.c_size_t(0)
    check(lib().m3_rmsnorm_bwd_workspace_size(rows, d, ctypes.byref(n)), "m3_rmsnorm_bwd_workspace_size")
    ws = torch.empty(max(n.value, 1), dtype=torch.uint8, device=x.device)
    check(lib().m3_rmsnorm_bwd(ptr(x), dtype_code(x.dtype), ptr(weight), dtype_code(weight.dtype),
                               ptr(rstd), ptr(grad), dtype_code(grad.dtype), ptr(dx), ptr(dweight),
                               ptr(ws), n.value, rows, d, stream_of(x)), "m3_rmsnorm_bwd")


# ---------------------------------------------------------------- training operators
def _bytes_of(name: str, *args) -> int:
    n = ctypes.c_size_t(0)
    check(getattr(lib(), name)(*args, ctypes.byref(n)), name)
    return n.value


def _workspace(nbytes: int, device) -> torch.Tensor | None:
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def swiglu_mlp_saved_bytes(rows: int, ff: int, dtype: torch.dtype) -> int:
    """m3_swiglu_mlp_saved_size, in arithmetic that a symbolic number of rows passes through: g and u in blocks of
    16 x 16 (24 bits each for bf16), then h with rows of whole 16 bytes."""
    size = dtype.itemsize
    wide = -(-ff * size // 16) * 16 // size
    kept = (rows + 15) // 16 * 16 * ((wide + 15) // 16 * 16) * (6 if size == 2 else 8)
    return (kept + 255) // 256 * 256 + (rows * wide * size + 255) // 256 * 256


def swiglu_mlp_fwd(x, w_gate, w_up, w_down, residual, scale, y, saved) -> None:
    """m3_swiglu_mlp_fwd on contiguous x (rows, d); allocates the workspace."""
    rows, d = x.shape
    dims = (rows, d, w_gate.shape[0], dtype_code(x.dtype))
    n = _bytes_of("m3_swiglu_mlp_fwd_workspace_size", *dims, int(saved is not None))
    ws = _workspace(n, x.device)
    check(lib().m3_swiglu_mlp_fwd(*dims, ptr(x), ptr(w_gate), ptr(w_up), ptr(w_down), ptr(residual), scale,
                                  ptr(y), ptr(saved), ptr(ws), n, stream_of(x)), "m3_swiglu_mlp_fwd")


def swiglu_mlp_bwd(x, w_gate, w_up, w_down, scale, saved, dy, dx, dw_gate, dw_up, dw_down) -> None:
    """m3_swiglu_mlp_bwd on contiguous (rows, d) tensors; allocates the workspace."""
    rows, d = x.shape
    dims = (rows, d, w_gate.shape[0], dtype_code(x.dtype))
    n = _bytes_of("m3_swiglu_mlp_bwd_workspace_size", *dims)
    ws = _workspace(n, x.device)
    check(lib().m3_swiglu_mlp_bwd(*dims, ptr(x), ptr(w_gate), ptr(w_up), ptr(w_down), scale, ptr(saved),
                                  ptr(dy), ptr(dx), ptr(dw_gate), ptr(dw_up), ptr(dw_down), ptr(ws), n,
                                  stream_of(x)), "m3_swiglu_mlp_bwd")


REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def linear_xent_fwd(hidden, weight, target, ignore_index, reduction, loss, lse, count) -> None:
    """m3_linear_xent_fwd on contiguous hidden (rows, d); allocates the workspace."""
    rows, d = hidden.shape
    dims = (rows, d, weight.shape[0], dtype_code(hidden.dtype))
    n = _bytes_of("m3_linear_xent_fwd_workspace_size", *dims)
    ws = _workspace(n, hidden.device)
    check(lib().m3_linear_xent_fwd(*dims, reduction, ptr(hidden), ptr(weight), ptr(target), ignore_index,
                                   ptr(loss), ptr(lse), ptr(count), ptr(ws), n, stream_of(hidden)),
          "m3_linear_xent_fwd")


def linear_xent_bwd(hidden, weight, target, ignore_index, reduction, lse, count, grad, dhidden,
                    dweight) -> None:
    """m3_linear_xent_bwd on contiguous hidden (rows, d); allocates the workspace."""
    rows, d = hidden.shape
    dims = (rows, d, weight.shape[0], dtype_code(hidden.dtype))
    n = _bytes_of("m3_linear_xent_bwd_workspace_size", *dims, int(dhidden is not None), int(dweight is not None))
    ws = _workspace(n, hidden.device)
    check(lib().m3_linear_xent_bwd(*dims, reduction, ptr(hidden), ptr(weight), ptr(target), ignore_index,
                                   ptr(lse), ptr(count), ptr(grad), ptr(dhidden), ptr(dweight), ptr(ws), n,
                                   stream_of(hidden)), "m3_linear_xent_bwd")


NORM_L2, NORM_MAX = 0, 1


def clip_grad_norm(ptrs, numel, dtypes, kind: int, max_norm: float | None, norm) -> None:
    """m3_clip_grad_norm on contiguous tensors, given as lists of addresses, sizes and dtype codes;
    max_norm None: the norm alone. Allocates the workspace."""
    n = len(ptrs)
    ptrs, numel, dtypes = array("Q", ptrs), array("q", numel), array("i", dtypes)
    p, k, d = (a.buffer_info()[0] for a in (ptrs, numel, dtypes))
    nbytes = _bytes_of("m3_clip_grad_norm_workspace_size", n, k, d)
    ws = _workspace(nbytes, norm.device)
    st = lib().m3_clip_grad_norm(n, p, k, d, kind, int(max_norm is not None),
                                 0.0 if max_norm is None else max_norm, ptr(norm), ptr(ws), nbytes,
                                 stream_of(norm))
    if st == M3_ERR_OVERLAP:
        raise ValueError("gradients that overlap in memory cannot be clipped in place")
    check(st, "m3_clip_grad_norm")


# ---------------------------------------------------------------- 4-bit serving
MX_FORMATS = {"e2m1": 0, "e4m3": 1}


def mx_padded(k: int) -> int:
    """Elements of a stored row of k microscaled values."""
    return -(-k // 128) * 128


def mx_row_bytes(k: int, fmt: str) -> int:
    return mx_padded(k) if fmt == "e4m3" else mx_padded(k) // 2


def mx_quantize(x, fmt: str, gated: bool, data, scales) -> None:
    """m3_mx_quantize on contiguous x (rows, k), or (rows, 2 k) when gated."""
    rows, k = x.shape
    st = lib().m3_mx_quantize(rows, k // 2 if gated else k, dtype_code(x.dtype), int(gated), MX_FORMATS[fmt],
                              x.data_ptr(), data.data_ptr(), scales.data_ptr(), stream_of(x))
    if st:
        check(st, "m3_mx_quantize")


def mx_dequantize(data, scales, fmt: str, out) -> None:
    """m3_mx_dequantize into contiguous out (rows, k)."""
    rows, k = out.shape
    st = lib().m3_mx_dequantize(rows, k, MX_FORMATS[fmt], dtype_code(out.dtype), data.data_ptr(), scales.data_ptr(),
                                out.data_ptr(), stream_of(out))
    if st:
        check(st, "m3_mx_dequantize")


def add_rmsnorm_fwd(x, residual, weight, scale: float, eps: float, total, y, rstd) -> None:
    """m3_add_rmsnorm_fwd on contiguous (rows, d) tensors."""
    rows, d = x.shape
    st = lib().m3_add_rmsnorm_fwd(rows, d, dtype_code(x.dtype), x.data_ptr(), residual.data_ptr(), weight.data_ptr(),
                                  scale, eps, total.data_ptr(), y.data_ptr(), ptr(rstd), stream_of(x))
    if st:
        check(st, "m3_add_rmsnorm_fwd")


def add_rmsnorm_mx(x, residual, weight, scale: float, eps: float, total, fmt: str, data, scales) -> None:
    """m3_add_rmsnorm_mx on contiguous (rows, d) tensors."""
    rows, d = x.shape
    st = lib().m3_add_rmsnorm_mx(rows, d, dtype_code(x.dtype), x.data_ptr(), ptr(residual), weight.data_ptr(), scale,
                                 eps, ptr(total), MX_FORMATS[fmt], data.data_ptr(), scales.data_ptr(), stream_of(x))
    if st:
        check(st, "m3_add_rmsnorm_mx")


@functools.lru_cache(maxsize=256)
def _add_rmsnorm_bwd_bytes(rows: int, d: int) -> int:
    return _bytes_of("m3_add_rmsnorm_bwd_workspace_size", rows, d)


def add_rmsnorm_bwd(total, weight, rstd, dtotal, dy, scale: float, dx, dresidual, dweight) -> None:
    """m3_add_rmsnorm_bwd on contiguous (rows, d) tensors; allocates the workspace."""
    rows, d = total.shape
    n = _add_rmsnorm_bwd_bytes(rows, d) if dweight is not None else 0
    ws = _workspace(n, total.device)
    check(lib().m3_add_rmsnorm_bwd(rows, d, dtype_code(total.dtype), ptr(total), ptr(weight), ptr(rstd), ptr(dtotal),
                                   ptr(dy), scale, ptr(dx), ptr(dresidual), ptr(dweight), ptr(ws), n,
                                   stream_of(total)), "m3_add_rmsnorm_bwd")


@functools.lru_cache(maxsize=1024)
def _mx_exact_bytes(rows: int, n: int, k: int) -> int:
    return _bytes_of("m3_mx_linear_exact_workspace_size", rows, n, k)


def mx_linear(x_data, x_scales, x_format: str, w_data, w_scales, k: int, residual, scale: float, out) -> None:
    """m3_mx_linear into contiguous out (rows, n), or m3_mx_linear_exact where it is the faster one; allocates its workspace."""
    rows, n = out.shape
    if out.dtype is torch.float32:
        size = _mx_exact_bytes(rows, n, k)
        if size:
            ws = _workspace(size, out.device)
            check(lib().m3_mx_linear_exact(rows, n, k, MX_FORMATS[x_format], x_data.data_ptr(), x_scales.data_ptr(), w_data.data_ptr(), w_scales.data_ptr(),
                                           ptr(residual), scale, out.data_ptr(), ptr(ws), size, stream_of(out)), "m3_mx_linear_exact")
            return
    st = lib().m3_mx_linear(rows, n, k, MX_FORMATS[x_format], dtype_code(out.dtype), x_data.data_ptr(), x_scales.data_ptr(),
                            w_data.data_ptr(), w_scales.data_ptr(), ptr(residual), scale, out.data_ptr(), stream_of(out))
    if st:
        check(st, "m3_mx_linear")


# What happens to a tensor before it is quantised and multiplied.
MX_AS_IS, MX_NORMED, MX_GATED = range(3)


def mx_linear_takes_tensor(rows: int, n: int, k: int, x_dtype: torch.dtype, out_dtype: torch.dtype, before: int) -> bool:
    return bool(lib().m3_mx_linear_takes_tensor(rows, n, k, dtype_code(x_dtype), dtype_code(out_dtype), before))


def mx_linear_tensor(x, norm_weight, eps: float, gated: bool, w_data, w_scales, residual, scale: float, out) -> None:
    """m3_mx_linear_tensor on contiguous x (rows, k), gated (rows, 2 k), into contiguous out (rows, n)."""
    rows, n = out.shape
    before = MX_GATED if gated else MX_AS_IS if norm_weight is None else MX_NORMED
    st = lib().m3_mx_linear_tensor(rows, n, x.shape[1] // 2 if gated else x.shape[1], dtype_code(x.dtype), dtype_code(out.dtype), before, x.data_ptr(),
                                   ptr(norm_weight), eps, w_data.data_ptr(), w_scales.data_ptr(), ptr(residual), scale, out.data_ptr(),
                                   stream_of(out))
    if st:
        check(st, "m3_mx_linear_tensor")


def sample_tokens(logits, u, temperature, top_k, top_p, min_p, token, logprob) -> None:
    """m3_sample_tokens on contiguous logits (rows, vocab); settings are numbers or tensors (rows,), fp32 or for
    top_k int32."""
    rows, vocab = logits.shape
    args = []
    for v in (temperature, top_k, top_p, min_p):
        args += [v.data_ptr(), 0] if isinstance(v, torch.Tensor) else [None, v]
    st = lib().m3_sample_tokens(rows, vocab, dtype_code(logits.dtype), logits.data_ptr(), u.data_ptr(), *args,
                                token.data_ptr(), ptr(logprob), stream_of(logits))
    if st:
        check(st, "m3_sample_tokens")
