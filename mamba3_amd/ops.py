"""torch.library custom ops over the C-ABI library (include/mamba3_amd.h).

Every native entry point the Python API uses is a registered op in the `mamba3_amd`
namespace with a fake (meta) kernel, and the differentiable ones with an autograd
formula, so that `torch.compile(fullgraph=True)` traces a KulaMamba layer, `chunked_ssd`
and `ssd_scan` without graph breaks, forward and backward (the reference keeps the same
property, mamba3/scan.py:5, tests/test_mamba3.py:584-616). The op bodies allocate
outputs and workspace with the caching allocator, take the current stream and call the
library through ctypes (`_native`); no op has a CPU or eager fallback.

Layer ops take the layer's shape as plain integers and its ten small parameters as
tensors in the order (A_log, D, dt_bias, B_norm.weight, C_norm.weight, B_bias, C_bias,
mimo_x, mimo_z, mimo_down); the kernels read fp32 copies of them, which are cached per
source tensor and version.
"""

from __future__ import annotations

import contextlib
import functools
import weakref
from collections import OrderedDict
from typing import Optional

import torch
from torch import _C
from torch.autograd import forward_ad as _forward_ad

from . import _native

NS = "mamba3_amd"

# ---------------------------------------------------------------------------- helpers
_F32_CACHE: "OrderedDict[tuple, list]" = OrderedDict()
_F32_CACHE_MAX = 256

def _cache_entry(params) -> list:
    """[LayerParams, fp32 tensors, weak refs] for the ten layer parameters. An entry is
    used only while every source tensor is the same live object at the same version."""
    # (an address names its device)
    key = (*[t.data_ptr() for t in params], *[t._version for t in params],
           *[t.dtype for t in params])
    hit = _F32_CACHE.get(key)
    if hit is not None:
        for r, t in zip(hit[2], params):
            if r() is not t:
                break
        else:
            _F32_CACHE.move_to_end(key)
            return hit
    with torch.no_grad():
        f32 = [t.detach().float().contiguous() for t in params]
    entry = [_native.LayerParams(*[t.data_ptr() for t in f32]), f32,
             [weakref.ref(t) for t in params]]
    _F32_CACHE[key] = entry
    while len(_F32_CACHE) > _F32_CACHE_MAX:
        _F32_CACHE.popitem(last=False)
    return entry


def _f32_params(params) -> tuple:
    """(LayerParams, fp32 tensors) for the ten layer parameters (cached)."""
    entry = _cache_entry(params)
    return entry[0], entry[1]


def _desc(batch, seqlen, nheads, headdim, d_state, mimo_rank, ngroups, trap, cplx, eps,
          dtype, row_stride) -> _native.LayerDesc:
    return _native.LayerDesc(batch, seqlen, nheads, headdim, d_state, mimo_rank, ngroups,
                             int(trap), int(cplx), _native.dtype_code(dtype), row_stride,
                             float(eps), 0)


def _state_shapes(B, nheads, headdim, d_state):
    return (B, nheads, headdim, d_state), (B, nheads, d_state // 2)


# ---------------------------------------------------------------------------- prefill
def _scratch(nbytes: int, device) -> torch.Tensor:
    return torch.empty(max(nbytes, 1), device=device, dtype=torch.uint8)


def _prefill_eager(proj, A_log, D, dt_bias, B_norm_w, C_norm_w, B_bias, C_bias, mimo_x, mimo_z,
                   mimo_down, dt_scale, nheads, headdim, d_state, mimo_rank, ngroups, trap, cplx,
                   eps, return_state):
    """m3_prefill_fwd: in_proj output (B,T,W) -> (y (B,T,H*P) in proj.dtype, h, angle,
    prev_BX), the states None without return_state."""
    _native.require_gpu(proj)
    proj = proj.contiguous()
    Bat, T, _ = proj.shape
    desc = _desc(Bat, T, nheads, headdim, d_state, mimo_rank, ngroups, trap, cplx, eps,
                 proj.dtype, proj.stride(-2))
    params = (A_log, D, dt_bias, B_norm_w, C_norm_w, B_bias, C_bias, mimo_x, mimo_z, mimo_down)
    pack, _ = _f32_params(params)
    dev = proj.device
    y = torch.empty(Bat, T, nheads * headdim, device=dev, dtype=proj.dtype)
    if return_state:
        hs, as_ = _state_shapes(Bat, nheads, headdim, d_state)
        h = torch.empty(hs, device=dev, dtype=torch.float32)
        angle = torch.empty(as_, device=dev, dtype=torch.float32)
        prev = torch.empty(hs, device=dev, dtype=torch.float32)
    else:
        h = angle = prev = None
    ws_bytes = _native.prefill_workspace_bytes(desc)
    try:
        ws = _scratch(ws_bytes, dev)
    except torch.OutOfMemoryError as e:
        oom = e
    else:
        _native.prefill_fwd(desc, pack, proj, dt_scale, y, h, angle, prev, ws, ws_bytes)
        return y, h, angle, prev
    # The kernels take a smaller workspace too (slices of the batch or the sequence).
    ws = None
    while ws is None and ws_bytes:
        ws_bytes = ws_bytes * 7 // 8
        try:
            ws = _scratch(ws_bytes, dev) if ws_bytes else None
        except torch.OutOfMemoryError:
            pass
    try:
        _native.prefill_fwd(desc, pack, proj, dt_scale, y, h, angle, prev, ws, ws_bytes)
    except _native.NativeError as e:
        if e.status == _native.M3_ERR_WORKSPACE:  # not even the operands fit
            raise oom from None
        raise
    return y, h, angle, prev


@torch.library.custom_op(f"{NS}::prefill", mutates_args=())
def prefill(proj: torch.Tensor, A_log: torch.Tensor, D: torch.Tensor, dt_bias: torch.Tensor,
            B_norm_w: torch.Tensor, C_norm_w: torch.Tensor, B_bias: torch.Tensor,
            C_bias: torch.Tensor, mimo_x: torch.Tensor, mimo_z: torch.Tensor,
            mimo_down: torch.Tensor, dt_scale: Optional[torch.Tensor], nheads: int,
            headdim: int, d_state: int, mimo_rank: int, ngroups: int, trap: bool, cplx: bool,
            eps: float, return_state: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor,
                                                     torch.Tensor]:
    """_prefill_eager as an op. Without return_state the three state tensors are empty."""
    out = _prefill_eager(proj, A_log, D, dt_bias, B_norm_w, C_norm_w, B_bias, C_bias, mimo_x,
                         mimo_z, mimo_down, dt_scale, nheads, headdim, d_state, mimo_rank, ngroups,
                         trap, cplx, eps, return_state)
    if return_state:
        return out
    # three distinct empty tensors: outputs of an op may not alias
    return (out[0], *(torch.empty(0, device=proj.device, dtype=torch.float32) for _ in range(3)))


@prefill.register_fake
def _(proj, A_log, D, dt_bias, B_norm_w, C_norm_w, B_bias, C_bias, mimo_x, mimo_z, mimo_down,
      dt_scale, nheads, headdim, d_state, mimo_rank, ngroups, trap, cplx, eps, return_state):
    Bat, T, _ = proj.shape
    y = proj.new_empty(Bat, T, nheads * headdim)
    if not return_state:
        e = proj.new_empty(0, dtype=torch.float32)
        return y, e, e.clone(), e.clone()
    hs, as_ = _state_shapes(Bat, nheads, headdim, d_state)
    return (y, proj.new_empty(hs, dtype=torch.float32), proj.new_empty(as_, dtype=torch.float32),
            proj.new_empty(hs, dtype=torch.float32))


# ------------------------------------------------------------ prefill for training
def _train_desc(proj, nheads, headdim, d_state, mimo_rank, ngroups, trap, cplx, eps):
    """fp32 descriptor of the training forward and of m3_layer_bwd: the forward keeps the
    intermediates the backward reads (M3_FLAG_FOR_BACKWARD)."""
    Bat, T, W = proj.shape
    desc = _desc(Bat, T, nheads, headdim, d_state, mimo_rank, ngroups, trap, cplx, eps,
                 torch.float32, W)
    desc.flags |= _native.M3_FLAG_FOR_BACKWARD
    return desc


@torch.library.custom_op(f"{NS}::prefill_train", mutates_args=())
def prefill_train(proj: torch.Tensor, A_log: torch.Tensor, D: torch.Tensor,
                  dt_bias: torch.Tensor, B_norm_w: torch.Tensor, C_norm_w: torch.Tensor,
                  B_bias: torch.Tensor, C_bias: torch.Tensor, mimo_x: torch.Tensor,
                  mimo_z: torch.Tensor, mimo_down: torch.Tensor,
                  dt_scale: Optional[torch.Tensor], nheads: int, headdim: int, d_state: int,
                  mimo_rank: int, ngroups: int, trap: bool, cplx: bool,
                  eps: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor,
                                       torch.Tensor]:
    """The prefill in fp32 arithmetic (bf16 inputs upcast) on the fp32 layer path, whose
    workspace (last output) holds the activations m3_layer_bwd differentiates through.
    Raises for shapes m3_layer_bwd does not cover."""
    _native.require_gpu(proj)
    proj32 = proj.detach().float().contiguous()
    desc = _train_desc(proj32, nheads, headdim, d_state, mimo_rank, ngroups, trap, cplx, eps)
    if not _native.layer_bwd_supported(desc):
        raise _native.NativeError(
            f"training through KulaMamba(d_state={d_state}, headdim={headdim}, "
            f"mimo_rank={mimo_rank}, ngroups={ngroups}) is not supported by m3_layer_bwd "
            "(the rank exceeds 8 or the shape exceeds the kernels' limits); "
            "run this layer without gradients")
    pack, _ = _f32_params((A_log, D, dt_bias, B_norm_w, C_norm_w, B_bias, C_bias, mimo_x,
                           mimo_z, mimo_down))
    Bat, T, _ = proj32.shape
    dev = proj.device
    ws_bytes = _native.prefill_workspace_bytes(desc)
    ws = torch.empty(max(ws_bytes, 1), device=dev, dtype=torch.uint8)
    y = torch.empty(Bat, T, nheads * headdim, device=dev, dtype=torch.float32)
    hs, as_ = _state_shapes(Bat, nheads, headdim, d_state)
    h = torch.empty(hs, device=dev, dtype=torch.float32)
    angle = torch.empty(as_, device=dev, dtype=torch.float32)
    prev = torch.empty(hs, device=dev, dtype=torch.float32)
    _native.prefill_fwd(desc, pack, proj32, dt_scale, y, h, angle, prev, ws, ws_bytes)
    return y.to(proj.dtype), h, angle, prev, ws


def _train_ws_bytes(proj, nheads, headdim, d_state, mimo_rank, ngroups, trap, cplx, eps) -> int:
    desc = _train_desc(proj, nheads, headdim, d_state, mimo_rank, ngroups, trap, cplx, eps)
    return max(_native.prefill_workspace_bytes(desc), 1)


@prefill_train.register_fake
def _(proj, A_log, D, dt_bias, B_norm_w, C_norm_w, B_bias, C_bias, mimo_x, mimo_z, mimo_down,
      dt_scale, nheads, headdim, d_state, mimo_rank, ngroups, trap, cplx, eps):
    Bat, T, _ = proj.shape
    hs, as_ = _state_shapes(Bat, nheads, headdim, d_state)
    n = _train_ws_bytes(proj, nheads, headdim, d_state, mimo_rank, ngroups, trap, cplx, eps)
    return (proj.new_empty(Bat, T, nheads * headdim), proj.new_empty(hs, dtype=torch.float32),
            proj.new_empty(as_, dtype=torch.float32), proj.new_empty(hs, dtype=torch.float32),
            proj.new_empty(n, dtype=torch.uint8))


@torch.library.custom_op(f"{NS}::layer_bwd", mutates_args=())
def layer_bwd(proj: torch.Tensor, A_log: torch.Tensor, D: torch.Tensor, dt_bias: torch.Tensor,
              B_norm_w: torch.Tensor, C_norm_w: torch.Tensor, B_bias: torch.Tensor,
              C_bias: torch.Tensor, mimo_x: torch.Tensor, mimo_z: torch.Tensor,
              mimo_down: torch.Tensor, dt_scale: Optional[torch.Tensor], fwd_ws: torch.Tensor,
              g_y: torch.Tensor, g_h: Optional[torch.Tensor], g_angle: Optional[torch.Tensor],
              g_prev: Optional[torch.Tensor], nheads: int, headdim: int, d_state: int,
              mimo_rank: int, ngroups: int, trap: bool, cplx: bool,
              eps: float) -> list[torch.Tensor]:
    """m3_layer_bwd: gradients of prefill_train's outputs with respect to proj (fp32), the
    ten parameters (fp32, their shapes) and dt_scale (fp32 (B,T,H); zeros when dt_scale
    is None)."""
    proj32 = proj.detach().float().contiguous()
    desc = _train_desc(proj32, nheads, headdim, d_state, mimo_rank, ngroups, trap, cplx, eps)
    params = (A_log, D, dt_bias, B_norm_w, C_norm_w, B_bias, C_bias, mimo_x, mimo_z, mimo_down)
    pack, f32 = _f32_params(params)

    def f32c(t):
        return None if t is None else t.float().contiguous()

    g_proj = torch.empty_like(proj32)
    grads = [torch.empty_like(t) for t in f32]
    Bat, T, _ = proj32.shape
    g_dts = torch.zeros(Bat, T, nheads, device=proj.device, dtype=torch.float32)
    _native.layer_bwd(desc, pack, proj32, dt_scale, fwd_ws, f32c(g_y), f32c(g_h), f32c(g_angle),
                      f32c(g_prev), g_proj,
                      _native.LayerParamGrads(*[t.data_ptr() for t in grads],
                                              g_dts.data_ptr() if dt_scale is not None else None))
    return [g_proj, *grads, g_dts]


@layer_bwd.register_fake
def _(proj, A_log, D, dt_bias, B_norm_w, C_norm_w, B_bias, C_bias, mimo_x, mimo_z, mimo_down,
      dt_scale, fwd_ws, g_y, g_h, g_angle, g_prev, nheads, headdim, d_state, mimo_rank, ngroups,
      trap, cplx, eps):
    params = (A_log, D, dt_bias, B_norm_w, C_norm_w, B_bias, C_bias, mimo_x, mimo_z, mimo_down)
    Bat, T, _ = proj.shape
    return [proj.new_empty(proj.shape, dtype=torch.float32),
            *[t.new_empty(t.shape, dtype=torch.float32) for t in params],
            proj.new_empty(Bat, T, nheads, dtype=torch.float32)]


def _prefill_train_setup(ctx, inputs, output):
    *tensors, dt_scale, nheads, headdim, d_state, mimo_rank, ngroups, trap, cplx, eps = inputs
    ctx.cfg = (nheads, headdim, d_state, mimo_rank, ngroups, trap, cplx, eps)
    ctx.has_scale = dt_scale is not None
    ctx.save_for_backward(*tensors, dt_scale, output[4])
    ctx.set_materialize_grads(False)


def _prefill_train_backward(ctx, g_y, g_h, g_angle, g_prev, g_ws):
    *tensors, dt_scale, ws = ctx.saved_tensors
    proj, params = tensors[0], tensors[1:]
    if g_y is None:
        g_y = proj.new_zeros(proj.shape[0], proj.shape[1], ctx.cfg[0] * ctx.cfg[1],
                             dtype=torch.float32)
    out = layer_bwd(proj, *params, dt_scale, ws, g_y, g_h, g_angle, g_prev, *ctx.cfg)
    g_proj, g_params, g_dts = out[0], out[1:11], out[11]
    grads = [g_proj.to(proj.dtype)] + [g.to(p.dtype) for g, p in zip(g_params, params)]
    grads.append(g_dts if ctx.has_scale else None)
    return (*grads, None, None, None, None, None, None, None, None)


prefill_train.register_autograd(_prefill_train_backward, setup_context=_prefill_train_setup)


# ---------------------------------------------------------------------------- step
def _step_eager(proj: torch.Tensor, A_log: torch.Tensor, D: torch.Tensor, dt_bias: torch.Tensor,
         B_norm_w: torch.Tensor, C_norm_w: torch.Tensor, B_bias: torch.Tensor,
         C_bias: torch.Tensor, mimo_x: torch.Tensor, mimo_z: torch.Tensor,
         mimo_down: torch.Tensor, dt_scale: Optional[torch.Tensor], h: torch.Tensor,
         prev_bx: torch.Tensor, angle: torch.Tensor, nheads: int, headdim: int, d_state: int,
         mimo_rank: int, ngroups: int, trap: bool, cplx: bool,
         eps: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """m3_step_fwd on one token per row: proj (B,W) and the state -> (y (B,H*P), new h,
    new prev_BX, new angle). The state comes back in new tensors (h and prev_BX fp32,
    angle in its input dtype). Its autograd formula is m3_step_bwd."""
    out = [torch.empty(proj.shape[0], nheads * headdim, device=proj.device, dtype=proj.dtype),
           torch.empty_like(h, dtype=torch.float32), torch.empty_like(prev_bx, dtype=torch.float32),
           torch.empty_like(angle)]
    step_into(proj, A_log, D, dt_bias, B_norm_w, C_norm_w, B_bias, C_bias, mimo_x, mimo_z,
              mimo_down, dt_scale, h, prev_bx, angle, *out, nheads, headdim, d_state,
              mimo_rank, ngroups, trap, cplx, eps)
    return tuple(out)


step = torch.library.custom_op(f"{NS}::step", _step_eager, mutates_args=())


@step.register_fake
def _(proj, A_log, D, dt_bias, B_norm_w, C_norm_w, B_bias, C_bias, mimo_x, mimo_z, mimo_down,
      dt_scale, h, prev_bx, angle, nheads, headdim, d_state, mimo_rank, ngroups, trap, cplx, eps):
    return (proj.new_empty(proj.shape[0], nheads * headdim), h.new_empty(h.shape, dtype=torch.float32),
            prev_bx.new_empty(prev_bx.shape, dtype=torch.float32), angle.new_empty(angle.shape))


@torch.library.custom_op(f"{NS}::step_bwd", mutates_args=())
def step_bwd(proj: torch.Tensor, A_log: torch.Tensor, D: torch.Tensor, dt_bias: torch.Tensor,
             B_norm_w: torch.Tensor, C_norm_w: torch.Tensor, B_bias: torch.Tensor,
             C_bias: torch.Tensor, mimo_x: torch.Tensor, mimo_z: torch.Tensor,
             mimo_down: torch.Tensor, dt_scale: Optional[torch.Tensor], h: torch.Tensor,
             prev_bx: torch.Tensor, angle: torch.Tensor, g_y: torch.Tensor,
             g_h: Optional[torch.Tensor], g_prev: Optional[torch.Tensor],
             g_angle: Optional[torch.Tensor], nheads: int, headdim: int, d_state: int,
             mimo_rank: int, ngroups: int, trap: bool, cplx: bool,
             eps: float) -> list[torch.Tensor]:
    """m3_step_bwd: gradients of step's outputs with respect to proj, the ten parameters,
    dt_scale (zeros when None) and the incoming h, prev_BX and angle, all fp32."""
    proj32 = proj.detach().float().contiguous()
    desc = _desc(proj32.shape[0], 1, nheads, headdim, d_state, mimo_rank, ngroups, trap, cplx,
                 eps, torch.float32, proj32.stride(0))
    if not _native.step_bwd_supported(desc):
        raise _native.NativeError(
            f"KulaMamba.step backward: this shape (d_state={d_state}, headdim={headdim}, "
            f"mimo_rank={mimo_rank}) is not supported by m3_step_bwd")
    params = (A_log, D, dt_bias, B_norm_w, C_norm_w, B_bias, C_bias, mimo_x, mimo_z, mimo_down)
    pack, f32 = _f32_params(params)

    def f32c(t):
        return None if t is None else t.detach().float().contiguous()

    g_proj = torch.zeros_like(proj32)
    grads = [torch.empty_like(t) for t in f32]
    g_dts = torch.zeros(proj32.shape[0], nheads, device=proj.device, dtype=torch.float32)
    h32, prev32, ang32 = f32c(h), f32c(prev_bx), f32c(angle)
    g_h_in, g_prev_in, g_ang_in = (torch.empty_like(h32), torch.empty_like(prev32),
                                   torch.empty_like(ang32))
    _native.step_bwd(desc, pack, proj32, f32c(dt_scale), h32, prev32, ang32, f32c(g_y), f32c(g_h),
                     f32c(g_prev), f32c(g_angle), g_proj, g_h_in, g_prev_in, g_ang_in,
                     _native.LayerParamGrads(*[t.data_ptr() for t in grads],
                                             g_dts.data_ptr() if dt_scale is not None else None))
    return [g_proj, *grads, g_dts, g_h_in, g_prev_in, g_ang_in]


@step_bwd.register_fake
def _(proj, A_log, D, dt_bias, B_norm_w, C_norm_w, B_bias, C_bias, mimo_x, mimo_z, mimo_down,
      dt_scale, h, prev_bx, angle, g_y, g_h, g_prev, g_angle, nheads, headdim, d_state,
      mimo_rank, ngroups, trap, cplx, eps):
    params = (A_log, D, dt_bias, B_norm_w, C_norm_w, B_bias, C_bias, mimo_x, mimo_z, mimo_down)
    f = torch.float32
    return [proj.new_empty(proj.shape, dtype=f), *[t.new_empty(t.shape, dtype=f) for t in params],
            proj.new_empty(proj.shape[0], nheads, dtype=f), h.new_empty(h.shape, dtype=f),
            prev_bx.new_empty(prev_bx.shape, dtype=f), angle.new_empty(angle.shape, dtype=f)]


def _step_setup(ctx, inputs, output):
    ctx.cfg = inputs[15:]
    ctx.has_scale = inputs[11] is not None
    ctx.save_for_backward(*inputs[:15])
    ctx.set_materialize_grads(False)


def _step_backward(ctx, g_y, g_h, g_prev, g_angle):
    proj, *rest = ctx.saved_tensors
    params, dt_scale, h, prev_bx, angle = rest[:10], rest[10], rest[11], rest[12], rest[13]
    if g_y is None:
        g_y = proj.new_zeros(proj.shape[0], ctx.cfg[0] * ctx.cfg[1], dtype=torch.float32)
    out = step_bwd(proj, *params, dt_scale, h, prev_bx, angle, g_y, g_h, g_prev, g_angle,
                   *ctx.cfg)
    g_proj, g_params, g_dts, g_hin, g_pin, g_ain = out[0], out[1:11], out[11], out[12], out[13], out[14]
    grads = [g_proj.to(proj.dtype)] + [g.to(p.dtype) for g, p in zip(g_params, params)]
    grads.append(g_dts if ctx.has_scale else None)
    grads += [g_hin.to(h.dtype), g_pin.to(prev_bx.dtype), g_ain.to(angle.dtype)]
    return (*grads, None, None, None, None, None, None, None, None)


step.register_autograd(_step_backward, setup_context=_step_setup)


def step_into(proj, A_log, D, dt_bias, B_norm_w, C_norm_w, B_bias, C_bias, mimo_x, mimo_z,
              mimo_down, dt_scale, h, prev_bx, angle, y_out, h_out, prev_out, angle_out,
              nheads, headdim, d_state, mimo_rank, ngroups, trap, cplx, eps) -> None:
    """m3_step_fwd into caller-owned outputs (which must not alias the inputs); used by the
    captured decode loop, which alternates two state buffer sets."""
    _native.require_gpu(proj, h, prev_bx, angle)
    proj = proj.contiguous()
    h = h.float().contiguous()
    prev_bx = prev_bx.float().contiguous()
    if angle.dtype not in (torch.float32, torch.bfloat16):
        angle = angle.float()
    angle = angle.contiguous()
    if angle_out.dtype != angle.dtype:
        raise TypeError("angle_out must have the dtype of the input angle")
    desc = _desc(proj.shape[0], 1, nheads, headdim, d_state, mimo_rank, ngroups, trap, cplx, eps,
                 proj.dtype, proj.stride(0))
    pack, _ = _f32_params((A_log, D, dt_bias, B_norm_w, C_norm_w, B_bias, C_bias, mimo_x,
                           mimo_z, mimo_down))
    _native.step_fwd(desc, pack, proj, dt_scale, h, prev_bx, angle, y_out, h_out, prev_out,
                     angle_out)


# ---------------------------------------------------------------------------- scan
@torch.library.custom_op(f"{NS}::scan_fwd", mutates_args=())
def scan_fwd(decay: torch.Tensor, h_chunk: torch.Tensor,
             h_init: Optional[torch.Tensor]) -> torch.Tensor:
    """m3_scan_fwd on fp32 (B,K,H) decay, (B,K,H,PN) h_chunk, (B,H,PN) h_init -> fp32 states."""
    _native.require_gpu(decay, h_chunk, h_init)
    decay = decay.float().contiguous()
    h_chunk = h_chunk.float().contiguous()
    if h_init is not None:
        h_init = h_init.float().contiguous()
    out = torch.empty_like(h_chunk)
    _native.scan_fwd(decay, h_chunk, h_init, out)
    return out


@scan_fwd.register_fake
def _(decay, h_chunk, h_init):
    return h_chunk.new_empty(h_chunk.shape, dtype=torch.float32)


@torch.library.custom_op(f"{NS}::scan_bwd", mutates_args=())
def scan_bwd(decay: torch.Tensor, h_states: torch.Tensor, grad: torch.Tensor,
             with_init: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """m3_scan_bwd -> (d_decay, d_chunk, d_h_init; the last empty without h_init)."""
    decay = decay.float().contiguous()
    grad = grad.float().contiguous()
    B, K, H, PN = h_states.shape
    d_decay = torch.empty_like(decay)
    d_chunk = torch.empty_like(h_states)
    d_init = torch.empty(B, H, PN, dtype=torch.float32, device=h_states.device) if with_init \
        else torch.empty(0, dtype=torch.float32, device=h_states.device)
    _native.scan_bwd(decay, h_states, grad, d_decay, d_chunk, d_init if with_init else None)
    return d_decay, d_chunk, d_init


@scan_bwd.register_fake
def _(decay, h_states, grad, with_init):
    B, K, H, PN = h_states.shape
    return (decay.new_empty(decay.shape, dtype=torch.float32),
            h_states.new_empty(h_states.shape, dtype=torch.float32),
            h_states.new_empty((B, H, PN) if with_init else (0,), dtype=torch.float32))


def _scan_setup(ctx, inputs, output):
    decay, h_chunk, h_init = inputs
    ctx.with_init = h_init is not None
    ctx.save_for_backward(decay, output)


def _scan_backward(ctx, grad):
    decay, states = ctx.saved_tensors
    d_decay, d_chunk, d_init = scan_bwd(decay, states, grad, ctx.with_init)
    return d_decay, d_chunk, (d_init if ctx.with_init else None)


scan_fwd.register_autograd(_scan_backward, setup_context=_scan_setup)


# ---------------------------------------------------------------------------- chunked SSD
@torch.library.custom_op(f"{NS}::chunked_fwd", mutates_args=())
def chunked_fwd(x_g: torch.Tensor, x_b: Optional[torch.Tensor], B_g: torch.Tensor,
                B_b: Optional[torch.Tensor], C: torch.Tensor, dt: torch.Tensor, A: torch.Tensor,
                D: torch.Tensor, x_raw: torch.Tensor,
                h_init: Optional[torch.Tensor]) -> tuple[torch.Tensor, torch.Tensor]:
    """m3_chunked_ssd_fwd: (y (B,T,H,P,R) in x_g.dtype, h_final (B,H,P,N) fp32). bf16 inputs
    of shapes the fp32-MFMA chunk kernels cover run on them in fp32 arithmetic."""
    Bat, T, H, P, R = x_g.shape
    N = B_g.shape[3]
    dtype = x_g.dtype
    calc = dtype
    if dtype != torch.float32 and _native.chunked_fwd_mfma_applies(Bat, T, H, P, N, R,
                                                                   x_b is not None):
        calc = torch.float32

    def prep(t):
        return None if t is None else t.to(calc).contiguous()

    xg, xb, Bg, Bb, Cc, dtc, xr = map(prep, (x_g, x_b, B_g, B_b, C, dt, x_raw))
    hi = None if h_init is None else h_init.reshape(Bat, H, P, N).float().contiguous()
    y = torch.empty(Bat, T, H, P, R, device=x_g.device, dtype=calc)
    h_final = torch.empty(Bat, H, P, N, device=x_g.device, dtype=torch.float32)
    _native.chunked_fwd(Bat, T, H, P, N, R, calc, xg, xb, Bg, Bb, Cc, dtc,
                        A.float().contiguous(), D.float().contiguous(), xr, hi, y, h_final, None)
    return y.to(dtype), h_final


@chunked_fwd.register_fake
def _(x_g, x_b, B_g, B_b, C, dt, A, D, x_raw, h_init):
    Bat, T, H, P, R = x_g.shape
    N = B_g.shape[3]
    return x_g.new_empty(x_g.shape), x_g.new_empty(Bat, H, P, N, dtype=torch.float32)


@torch.library.custom_op(f"{NS}::chunked_bwd", mutates_args=())
def chunked_bwd(x_g: torch.Tensor, x_b: Optional[torch.Tensor], B_g: torch.Tensor,
                B_b: Optional[torch.Tensor], C: torch.Tensor, dt: torch.Tensor, A: torch.Tensor,
                D: torch.Tensor, x_raw: torch.Tensor, h_init: Optional[torch.Tensor],
                dy: torch.Tensor, dh_final: Optional[torch.Tensor]) -> list[torch.Tensor]:
    """m3_chunked_ssd_bwd (fp32): [dx_g, dx_b, dB_g, dB_b, dC, ddt, dA, dD, dx_raw, dh_init];
    dx_b / dB_b / dh_init are empty when the input is None."""
    Bat, T, H, P, R = x_g.shape
    N = B_g.shape[3]
    dev = x_g.device

    def f32(t):
        return None if t is None else t.float().contiguous()

    def new(shape):
        return torch.empty(shape, device=dev, dtype=torch.float32)

    beta = x_b is not None
    g = [new(x_g.shape), new(x_b.shape) if beta else None, new(B_g.shape),
         new(B_b.shape) if beta else None, new(C.shape), new((Bat, T, H)), new((H,)), new((H,)),
         new(x_raw.shape), new((Bat, H, P, N)) if h_init is not None else None]
    hi = None if h_init is None else f32(h_init.reshape(Bat, H, P, N))
    _native.chunked_bwd(Bat, T, H, P, N, R, f32(x_g), f32(x_b), f32(B_g), f32(B_b), f32(C),
                        f32(dt), f32(A), f32(D), f32(x_raw), hi, f32(dy), f32(dh_final), *g)
    return [torch.empty(0, device=dev, dtype=torch.float32) if t is None else t for t in g]


@chunked_bwd.register_fake
def _(x_g, x_b, B_g, B_b, C, dt, A, D, x_raw, h_init, dy, dh_final):
    Bat, T, H, P, R = x_g.shape
    N = B_g.shape[3]

    def new(shape):
        return x_g.new_empty(shape, dtype=torch.float32)

    e = (0,)
    return [new(x_g.shape), new(x_b.shape if x_b is not None else e), new(B_g.shape),
            new(B_b.shape if B_b is not None else e), new(C.shape), new((Bat, T, H)), new((H,)),
            new((H,)), new(x_raw.shape), new((Bat, H, P, N) if h_init is not None else e)]


def _chunked_setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs)
    ctx.set_materialize_grads(False)


def _chunked_backward(ctx, dy, dh_final):
    ins = ctx.saved_tensors
    x_g = ins[0]
    if dy is None:
        dy = torch.zeros(x_g.shape, device=x_g.device, dtype=torch.float32)
    g = chunked_bwd(*ins, dy, dh_final)
    out = []
    for grad, like in zip(g, ins):
        out.append(None if like is None else grad.to(like.dtype).reshape(like.shape))
    return tuple(out)


chunked_fwd.register_autograd(_chunked_backward, setup_context=_chunked_setup)


def layer_args(layer) -> tuple:
    """The integer / flag arguments of the layer ops for a KulaMamba module."""
    return (layer.nheads, layer.headdim, layer.d_state, layer.mimo_rank, layer.ngroups,
            bool(layer.use_trapezoidal), bool(layer.use_complex_ssm), float(layer.B_norm.eps))


# ---------------------------------------------------------------------------- RMSNorm
def _rmsnorm_eager(x: torch.Tensor, weight: torch.Tensor, eps: float, keep: bool = False):
    """m3_rmsnorm_fwd over the last dimension of x: y in the promotion of x's and the weight's
    dtypes, and with `keep` rstd (rows,) fp32 (else None)."""
    _native.require_gpu(x, weight)
    x2 = x.reshape(-1, x.shape[-1]).contiguous()
    y = torch.empty(x2.shape, device=x.device,
                    dtype=x.dtype if x.dtype == weight.dtype
                    else torch.promote_types(x.dtype, weight.dtype))
    rstd = torch.empty(x2.shape[0], device=x.device, dtype=torch.float32) if keep else None
    _native.rmsnorm_fwd(x2, weight.contiguous(), y, rstd, eps)
    return y.view(x.shape), rstd


@torch.library.custom_op(f"{NS}::rmsnorm", mutates_args=())
def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    """m3_rmsnorm_fwd over the last dimension of x: (y in the promotion of x's and the
    weight's dtypes, rstd (rows,) fp32)."""
    return _rmsnorm_eager(x, weight, eps, True)


@rmsnorm.register_fake
def _(x, weight, eps):
    rows = x.numel() // x.shape[-1]
    return (x.new_empty(x.shape, dtype=torch.promote_types(x.dtype, weight.dtype)),
            x.new_empty(rows, dtype=torch.float32))


@torch.library.custom_op(f"{NS}::rmsnorm_bwd", mutates_args=())
def rmsnorm_bwd(x: torch.Tensor, weight: torch.Tensor, rstd: torch.Tensor,
                grad: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """m3_rmsnorm_bwd: (dL/dx in x's dtype, dL/dweight in the weight's dtype)."""
    d = x.shape[-1]
    x2 = x.reshape(-1, d).contiguous()
    g2 = grad.reshape(-1, d).contiguous().to(torch.promote_types(x.dtype, weight.dtype))
    dx = torch.empty_like(x2)
    dw = torch.empty_like(weight.contiguous())
    _native.rmsnorm_bwd(x2, weight.contiguous(), rstd, g2, dx, dw)
    return dx.reshape(x.shape), dw


@rmsnorm_bwd.register_fake
def _(x, weight, rstd, grad):
    return x.new_empty(x.shape), weight.new_empty(weight.shape)


def _rmsnorm_setup(ctx, inputs, output):
    x, weight, eps = inputs
    ctx.save_for_backward(x, weight, output[1])


def _rmsnorm_backward(ctx, g_y, g_rstd):
    x, weight, rstd = ctx.saved_tensors
    dx, dw = rmsnorm_bwd(x, weight, rstd, g_y)
    return dx, dw, None


rmsnorm.register_autograd(_rmsnorm_backward, setup_context=_rmsnorm_setup)


# ---------------------------------------------------------------- small-batch projections
def small_proj_usable(x: torch.Tensor, *weights, norm: bool = False) -> bool:
    """True when m3_small_linear / m3_small_swiglu take x (m, k) with these weights (norm
    weight and projection weights): bf16, at most 8 rows, k a multiple of 64 that fits their
    LDS (with the norm weight when `norm`), contiguous 16-byte aligned rows, and no autograd
    to record (the kernels have no backward)."""
    if torch.compiler.is_compiling() or x.dim() != 2 or x.dtype != torch.bfloat16:
        return False
    if not _native.small_proj_ok(x.shape[0], x.shape[1], norm):
        return False
    grad = torch.is_grad_enabled()
    for t in (x, *weights):
        if t is None or t.dtype != torch.bfloat16 or not t.is_cuda or not t.is_contiguous():
            return False
        if t.data_ptr() % 16 != 0 or (grad and t.requires_grad):
            return False
    return True


def _small_linear_eager(x: torch.Tensor, norm_w: Optional[torch.Tensor], eps: float, weight: torch.Tensor,
                 residual: Optional[torch.Tensor], scale: float) -> torch.Tensor:
    """m3_small_linear: [residual +] scale * (n W^T), n = RMSNorm(x; norm_w) or x, for bf16
    x (m <= 8, k) (check with small_proj_usable); no backward."""
    _native.require_gpu(x, weight)
    out = torch.empty(x.shape[0], weight.shape[0], device=x.device, dtype=torch.bfloat16)
    res = None if residual is None else residual.contiguous()
    _native.small_linear(x, norm_w, eps, weight, res, scale, out)
    return out


small_linear = torch.library.custom_op(f"{NS}::small_linear", _small_linear_eager, mutates_args=())


@small_linear.register_fake
def _(x, norm_w, eps, weight, residual, scale):
    return x.new_empty(x.shape[0], weight.shape[0])


def _small_swiglu_eager(x: torch.Tensor, norm_w: Optional[torch.Tensor], eps: float,
                 w_gate: torch.Tensor, w_up: torch.Tensor) -> torch.Tensor:
    """m3_small_swiglu: silu(n W_gate^T) * (n W_up^T), n = RMSNorm(x; norm_w) or x, for bf16
    x (m <= 8, k); no backward."""
    _native.require_gpu(x, w_gate, w_up)
    out = torch.empty(x.shape[0], w_gate.shape[0], device=x.device, dtype=torch.bfloat16)
    _native.small_swiglu(x, norm_w, eps, w_gate, w_up, out)
    return out


small_swiglu = torch.library.custom_op(f"{NS}::small_swiglu", _small_swiglu_eager, mutates_args=())


@small_swiglu.register_fake
def _(x, norm_w, eps, w_gate, w_up):
    return x.new_empty(x.shape[0], w_gate.shape[0])


def _silu_mul_eager(gate_up: torch.Tensor, d_ff: int) -> torch.Tensor:
    """m3_silu_mul: silu(gate_up[..., :d_ff]) * gate_up[..., d_ff:2 d_ff] for bf16 rows (the
    output of one GEMM over [w_gate; w_up]); no backward."""
    _native.require_gpu(gate_up)
    g2 = gate_up.reshape(-1, gate_up.shape[-1])
    if g2.stride(-1) != 1:
        g2 = g2.contiguous()
    out = torch.empty(g2.shape[0], d_ff, device=gate_up.device, dtype=torch.bfloat16)
    _native.silu_mul(g2, d_ff, out)
    return out.view(*gate_up.shape[:-1], d_ff)


silu_mul = torch.library.custom_op(f"{NS}::silu_mul", _silu_mul_eager, mutates_args=())


@silu_mul.register_fake
def _(gate_up, d_ff):
    return gate_up.new_empty(*gate_up.shape[:-1], d_ff)


# ---------------------------------------------------------------- training operators
def _flat(t: torch.Tensor) -> torch.Tensor:
    """t as contiguous, 16-byte aligned rows of its last dimension."""
    if t.dim() != 2 or not t.is_contiguous():
        t = t.detach().reshape(-1, t.shape[-1]).contiguous()
    return t if t.data_ptr() % 16 == 0 else t.detach().clone()


def on_device(t: torch.Tensor):
    """t's device as the current one (kernels are launched, and workspaces allocated, there)."""
    return _NO_SWITCH if _C._cuda_getDevice() == t.get_device() else torch.cuda.device(t.device)


_NO_SWITCH = contextlib.nullcontext()


def check_alike(what: str, *tensors: torch.Tensor) -> None:
    """Raises unless the tensors share a dtype that the kernels take and a GPU."""
    first = tensors[0]
    _native.dtype_code(first.dtype)
    for t in tensors[1:]:
        if t.dtype != first.dtype:
            raise TypeError(f"{what} takes tensors of one dtype, got {first.dtype} and {t.dtype}")
        if t.device != first.device:
            raise ValueError(f"{what} takes tensors on one GPU, got {first.device} and {t.device}")
    _native.require_gpu(first)


def autocast(*tensors):
    """The tensors in the type that torch.autocast runs products in, where that is bf16."""
    if not torch.is_autocast_enabled("cuda") or torch.get_autocast_dtype("cuda") is not torch.bfloat16:
        return tensors
    return tuple(t.to(torch.bfloat16) for t in tensors)


def _swiglu_mlp_eager(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
                      residual: Optional[torch.Tensor], scale: float,
                      keep: bool) -> tuple[torch.Tensor, Optional[torch.Tensor]]:
    """m3_swiglu_mlp_fwd over the last dimension of x: y in x's shape and, with `keep`, what the
    backward reads (else None)."""
    _native.require_gpu(x, w_gate, w_up, w_down, residual)
    with on_device(x):
        x2 = _flat(x)
        y = torch.empty(x2.shape, device=x.device, dtype=x.dtype)
        n = _native.swiglu_mlp_saved_bytes(x2.shape[0], w_gate.shape[0], x.dtype) if keep else 0
        saved = torch.empty(n, device=x.device, dtype=torch.uint8) if keep else None
        _native.swiglu_mlp_fwd(x2, _flat(w_gate), _flat(w_up), _flat(w_down),
                               None if residual is None else _flat(residual), scale, y, saved)
    return y.view(x.shape), saved


@torch.library.custom_op(f"{NS}::swiglu_mlp", mutates_args=())
def swiglu_mlp(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
               residual: Optional[torch.Tensor], scale: float,
               keep: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """_swiglu_mlp_eager as an op; the second output is empty without `keep`."""
    y, saved = _swiglu_mlp_eager(x, w_gate, w_up, w_down, residual, scale, keep)
    return y, x.new_empty(0, dtype=torch.uint8) if saved is None else saved


@swiglu_mlp.register_fake
def _(x, w_gate, w_up, w_down, residual, scale, keep):
    n = _native.swiglu_mlp_saved_bytes(x.numel() // x.shape[-1], w_gate.shape[0], x.dtype) if keep else 0
    return x.new_empty(x.shape), x.new_empty(n, dtype=torch.uint8)


def _swiglu_mlp_bwd_eager(x, w_gate, w_up, w_down, scale, saved, dy, want) -> list:
    """m3_swiglu_mlp_bwd: gradients of x, w_gate, w_up and w_down in their shapes, None for those that
    `want` leaves out."""
    with on_device(x):
        out = [torch.empty(t.shape, device=x.device, dtype=x.dtype) if w else None
               for t, w in zip((x, w_gate, w_up, w_down), want)]
        dy2 = _flat(dy if dy.dtype == x.dtype else dy.to(x.dtype))
        _native.swiglu_mlp_bwd(_flat(x), _flat(w_gate), _flat(w_up), _flat(w_down), scale, saved, dy2, *out)
    return out


@torch.library.custom_op(f"{NS}::swiglu_mlp_bwd", mutates_args=())
def swiglu_mlp_bwd(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
                   scale: float, saved: torch.Tensor, dy: torch.Tensor,
                   want: list[bool]) -> list[torch.Tensor]:
    """_swiglu_mlp_bwd_eager as an op; gradients that `want` leaves out are empty."""
    out = _swiglu_mlp_bwd_eager(x, w_gate, w_up, w_down, scale, saved, dy, want)
    return [x.new_empty(0) if t is None else t for t in out]


@swiglu_mlp_bwd.register_fake
def _(x, w_gate, w_up, w_down, scale, saved, dy, want):
    return [x.new_empty(t.shape if w else (0,)) for t, w in zip((x, w_gate, w_up, w_down), want)]


def _swiglu_mlp_setup(ctx, inputs, output):
    *tensors, _, scale, keep = inputs
    ctx.scale, ctx.keep = scale, keep
    ctx.save_for_backward(*tensors, output[1])
    ctx.set_materialize_grads(False)


def _swiglu_mlp_backward(ctx, dy, _):
    if dy is None:
        return (None,) * 7
    if not ctx.keep:
        raise RuntimeError("swiglu_mlp was run without keeping what its backward reads")
    *tensors, saved = ctx.saved_tensors
    want = list(ctx.needs_input_grad[:4])
    g = swiglu_mlp_bwd(*tensors, ctx.scale, saved, dy, want) if any(want) else [None] * 4
    return (*[t if w else None for t, w in zip(g, want)], dy if ctx.needs_input_grad[4] else None, None, None)


swiglu_mlp.register_autograd(_swiglu_mlp_backward, setup_context=_swiglu_mlp_setup)


class _SwigluMlp(torch.autograd.Function):
    """swiglu_mlp under eager autograd: the same calls without the dispatcher's host time, which is
    longer than the kernels' time for small inputs."""

    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, residual, scale):
        y, saved = _swiglu_mlp_eager(x, w_gate, w_up, w_down, residual, scale, True)
        ctx.scale = scale
        ctx.save_for_backward(x, w_gate, w_up, w_down, saved)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        *tensors, saved = ctx.saved_tensors
        want = ctx.needs_input_grad
        g = _swiglu_mlp_bwd_eager(*tensors, ctx.scale, saved, dy, want[:4]) if any(want[:4]) else [None] * 4
        return (*g, dy if want[4] else None, None)


def _linear_xent_eager(hidden: torch.Tensor, weight: torch.Tensor, target: torch.Tensor,
                       ignore_index: int,
                       reduction: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """m3_linear_xent_fwd: (loss, fp32, of target's shape or a scalar; lse (rows,); count (1,))."""
    _native.require_gpu(hidden, weight, target)
    with on_device(hidden):
        h2, t1 = _flat(hidden), target.reshape(-1).contiguous()
        new = lambda *s: torch.empty(s, device=hidden.device, dtype=torch.float32)  # noqa: E731
        loss = new(*target.shape) if reduction == 0 else new()
        lse, count = new(h2.shape[0]), new(1)
        _native.linear_xent_fwd(h2, _flat(weight), t1, ignore_index, reduction, loss, lse, count)
    return loss, lse, count


linear_xent = torch.library.custom_op(f"{NS}::linear_xent", _linear_xent_eager, mutates_args=())


@linear_xent.register_fake
def _(hidden, weight, target, ignore_index, reduction):
    f = torch.float32
    return (hidden.new_empty(target.shape if reduction == 0 else (), dtype=f),
            hidden.new_empty(target.numel(), dtype=f), hidden.new_empty(1, dtype=f))


def _linear_xent_bwd_eager(hidden, weight, target, ignore_index, reduction, lse, count, grad, want) -> list:
    """m3_linear_xent_bwd: gradients of hidden and weight, None for those that `want` leaves out."""
    with on_device(hidden):
        out = [torch.empty(t.shape, device=t.device, dtype=t.dtype) if w else None
               for t, w in zip((hidden, weight), want)]
        if grad.dtype != torch.float32 or not grad.is_contiguous():
            grad = grad.float().contiguous()
        _native.linear_xent_bwd(_flat(hidden), _flat(weight), target.reshape(-1).contiguous(), ignore_index,
                                reduction, lse, count, grad, *out)
    return out


@torch.library.custom_op(f"{NS}::linear_xent_bwd", mutates_args=())
def linear_xent_bwd(hidden: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, ignore_index: int,
                    reduction: int, lse: torch.Tensor, count: torch.Tensor, grad: torch.Tensor,
                    want: list[bool]) -> list[torch.Tensor]:
    """_linear_xent_bwd_eager as an op; gradients that `want` leaves out are empty."""
    out = _linear_xent_bwd_eager(hidden, weight, target, ignore_index, reduction, lse, count, grad, want)
    return [hidden.new_empty(0) if t is None else t for t in out]


@linear_xent_bwd.register_fake
def _(hidden, weight, target, ignore_index, reduction, lse, count, grad, want):
    return [hidden.new_empty(t.shape if w else (0,)) for t, w in zip((hidden, weight), want)]


def _linear_xent_setup(ctx, inputs, output):
    hidden, weight, target, ctx.ignore_index, ctx.reduction = inputs
    ctx.save_for_backward(hidden, weight, target, output[1], output[2])
    ctx.set_materialize_grads(False)


def _linear_xent_backward(ctx, g_loss, g_lse, g_count):
    if g_loss is None:
        return (None,) * 5
    hidden, weight, target, lse, count = ctx.saved_tensors
    want = list(ctx.needs_input_grad[:2])
    g = linear_xent_bwd(hidden, weight, target, ctx.ignore_index, ctx.reduction, lse, count, g_loss, want)
    return (*[t if w else None for t, w in zip(g, want)], None, None, None)


linear_xent.register_autograd(_linear_xent_backward, setup_context=_linear_xent_setup)


class _LinearXent(torch.autograd.Function):
    """linear_xent under eager autograd, without the dispatcher's host time."""

    @staticmethod
    def forward(ctx, hidden, weight, target, ignore_index, reduction):
        loss, lse, count = _linear_xent_eager(hidden, weight, target, ignore_index, reduction)
        ctx.cfg = ignore_index, reduction
        ctx.save_for_backward(hidden, weight, target, lse, count)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        hidden, weight, target, lse, count = ctx.saved_tensors
        g = _linear_xent_bwd_eager(hidden, weight, target, *ctx.cfg, lse, count, grad, ctx.needs_input_grad[:2])
        return (*g, None, None, None)


# ---------------------------------------------------------------- eager calls
# What a direct call may be given: a subclass's own dispatch has to see it.
_PLAIN = frozenset((torch.Tensor, torch.nn.Parameter, type(None)))


def _direct(*tensors) -> bool:
    """Eager calls with autograd off bypass the dispatcher: its per-call host time (16 us for
    the prefill op) is what a per-token decode loop and a short prompt wait on. Traced calls,
    calls under autograd, a dispatch or function mode, a functorch transform or forward-mode
    AD, and calls with a tensor subclass among `tensors` (all tensor arguments of the op) go
    through the registered ops and their formulas."""
    return not _is_grad_enabled() and _plain(*tensors)


def _plain(*tensors) -> bool:
    """_direct's conditions but for autograd: what a torch.autograd.Function may stand in for."""
    if _is_compiling():
        return False
    if (_in_dispatch_mode() or _in_function_mode() or _tracing_state() is not None
            or _functorch_stack() is not None or _forward_ad._current_level >= 0):
        return False
    return _PLAIN.issuperset(map(type, tensors))


_is_grad_enabled, _is_compiling = torch.is_grad_enabled, torch.compiler.is_compiling
# torch's private counters of the modes and transforms that a direct call would pass by; on a
# torch version that lacks one of them every call goes through the ops.
try:
    _in_dispatch_mode, _in_function_mode = _C._len_torch_dispatch_stack, _C._len_torch_function_stack
    _tracing_state, _functorch_stack = _C._get_tracing_state, _C._functorch.peek_interpreter_stack
    _forward_ad._current_level
except AttributeError:
    def _plain(*tensors) -> bool:
        return False


def prefill_fast(*args):
    return (_prefill_eager if _direct(*args[:12]) else prefill)(*args)


def step_fast(*args):
    return (_step_eager if _direct(*args[:15]) else step)(*args)


def small_linear_fast(x, norm_w, eps, weight, residual, scale):
    fn = _small_linear_eager if _direct(x, norm_w, weight, residual) else small_linear
    return fn(x, norm_w, eps, weight, residual, scale)


def small_swiglu_fast(x, norm_w, eps, w_gate, w_up):
    fn = _small_swiglu_eager if _direct(x, norm_w, w_gate, w_up) else small_swiglu
    return fn(x, norm_w, eps, w_gate, w_up)


def silu_mul_fast(gate_up, d_ff):
    return (_silu_mul_eager if _direct(gate_up) else silu_mul)(gate_up, d_ff)


def rmsnorm_fast(x, weight, eps):
    return (_rmsnorm_eager if _direct(x, weight) else rmsnorm)(x, weight, eps)[0]


def swiglu_mlp_fast(x, w_gate, w_up, w_down, residual, scale, keep):
    if not _plain(x, w_gate, w_up, w_down, residual):
        return swiglu_mlp(x, w_gate, w_up, w_down, residual, scale, keep)[0]
    if keep:
        return _SwigluMlp.apply(x, w_gate, w_up, w_down, residual, scale)
    return _swiglu_mlp_eager(x, w_gate, w_up, w_down, residual, scale, False)[0]


def linear_xent_fast(hidden, weight, target, ignore_index, reduction):
    if not _plain(hidden, weight, target):
        return linear_xent(hidden, weight, target, ignore_index, reduction)[0]
    if _is_grad_enabled() and (hidden.requires_grad or weight.requires_grad):
        return _LinearXent.apply(hidden, weight, target, ignore_index, reduction)
    return _linear_xent_eager(hidden, weight, target, ignore_index, reduction)[0]


# ---------------------------------------------------------------- 4-bit serving
def _rows_of(t: torch.Tensor) -> torch.Tensor:
    """t as contiguous rows of its last dimension; these kernels take them at any alignment."""
    return t if t.dim() == 2 and t.is_contiguous() else t.detach().reshape(-1, t.shape[-1]).contiguous()


def _mx_empty(rows: int, k: int, fmt: str, like: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Room for (rows, k) microscaled values: (data, scales)."""
    kp = _native.mx_padded(k)
    return (like.new_empty((rows, kp if fmt == "e4m3" else kp // 2), dtype=torch.uint8),
            like.new_empty((rows, kp // 32), dtype=torch.uint8))


def _mx_quantize_eager(x: torch.Tensor, fmt: str, gated: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """m3_mx_quantize over the last dimension of x: (data, scales), one row for each of x's."""
    _native.require_gpu(x)
    with on_device(x):
        x2 = _rows_of(x)
        rows, k = x2.shape
        out = _mx_empty(rows, k // 2 if gated else k, fmt, x2)
        if rows:
            _native.mx_quantize(x2, fmt, gated, *out)
    return out


mx_quantize = torch.library.custom_op(f"{NS}::mx_quantize", _mx_quantize_eager, mutates_args=())


@mx_quantize.register_fake
def _(x, fmt, gated):
    k = x.shape[-1] // 2 if gated else x.shape[-1]
    return _mx_empty(x.numel() // x.shape[-1], k, fmt, x)


def _mx_dequantize_eager(data: torch.Tensor, scales: torch.Tensor, fmt: str, k: int, dtype: torch.dtype) -> torch.Tensor:
    """m3_mx_dequantize: (rows, k) in `dtype`."""
    _native.require_gpu(data, scales)
    with on_device(data):
        rows = data.shape[0]
        out = data.new_empty((rows, k), dtype=dtype)
        if rows:
            _native.mx_dequantize(data, scales, fmt, out)
    return out


mx_dequantize = torch.library.custom_op(f"{NS}::mx_dequantize", _mx_dequantize_eager, mutates_args=())


@mx_dequantize.register_fake
def _(data, scales, fmt, k, dtype):
    return data.new_empty((data.shape[0], k), dtype=dtype)


def _add_rmsnorm_eager(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, scale: float,
                       eps: float, keep: bool = True) -> tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """m3_add_rmsnorm_fwd over the last dimension: (total, y, and with `keep` rstd (rows,) fp32)."""
    _native.require_gpu(x, residual, weight)
    with on_device(x):
        x2 = _rows_of(x)
        total, y = torch.empty_like(x2), torch.empty_like(x2)
        rstd = torch.empty(x2.shape[0], device=x.device, dtype=torch.float32) if keep else None
        _native.add_rmsnorm_fwd(x2, _rows_of(residual), weight.contiguous(), scale, eps, total, y, rstd)
    return (total, y, rstd) if x.dim() == 2 else (total.view(x.shape), y.view(x.shape), rstd)


@torch.library.custom_op(f"{NS}::add_rmsnorm", mutates_args=())
def add_rmsnorm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, scale: float,
                eps: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """_add_rmsnorm_eager as an op."""
    return _add_rmsnorm_eager(x, residual, weight, scale, eps)


@add_rmsnorm.register_fake
def _(x, residual, weight, scale, eps):
    return x.new_empty(x.shape), x.new_empty(x.shape), x.new_empty(x.numel() // x.shape[-1], dtype=torch.float32)


def _add_rmsnorm_bwd_eager(total, weight, rstd, dtotal, dy, scale, want) -> list:
    """m3_add_rmsnorm_bwd: gradients of x, residual and weight, None for those that `want` leaves out."""
    with on_device(total):
        t2, w1 = _rows_of(total), weight.contiguous()
        out = [torch.empty_like(t) if w else None for t, w in zip((t2, t2, w1), want)]
        dy = _rows_of(dy if dy.dtype == total.dtype else dy.to(total.dtype))
        if dtotal is not None:
            dtotal = _rows_of(dtotal if dtotal.dtype == total.dtype else dtotal.to(total.dtype))
        _native.add_rmsnorm_bwd(t2, w1, rstd, dtotal, dy, scale, *out)
    if total.dim() != 2:
        out[:2] = [None if t is None else t.view(total.shape) for t in out[:2]]
    return out


@torch.library.custom_op(f"{NS}::add_rmsnorm_bwd", mutates_args=())
def add_rmsnorm_bwd(total: torch.Tensor, weight: torch.Tensor, rstd: torch.Tensor, dtotal: Optional[torch.Tensor],
                    dy: torch.Tensor, scale: float, want: list[bool]) -> list[torch.Tensor]:
    """_add_rmsnorm_bwd_eager as an op; gradients that `want` leaves out are empty."""
    out = _add_rmsnorm_bwd_eager(total, weight, rstd, dtotal, dy, scale, want)
    return [total.new_empty(0) if t is None else t for t in out]


@add_rmsnorm_bwd.register_fake
def _(total, weight, rstd, dtotal, dy, scale, want):
    return [t.new_empty(t.shape if w else (0,)) for t, w in zip((total, total, weight), want)]


def _add_rmsnorm_grads(bwd, total, weight, rstd, scale, want, dtotal, dy):
    """The three gradients; either output's may be None."""
    if dy is None:
        # the norm's output is unused: the sum alone
        if dtotal is None:
            return None, None, None
        return (dtotal * scale if want[0] else None, dtotal if want[1] else None,
                torch.zeros_like(weight) if want[2] else None)
    if not any(want):
        return None, None, None
    out = bwd(total, weight, rstd, dtotal, dy, scale, list(want))
    return tuple(t if w else None for t, w in zip(out, want))


def _add_rmsnorm_setup(ctx, inputs, output):
    _, _, weight, ctx.scale, _ = inputs
    ctx.save_for_backward(output[0], weight, output[2])
    ctx.set_materialize_grads(False)


def _add_rmsnorm_backward(ctx, dtotal, dy, _):
    grads = _add_rmsnorm_grads(add_rmsnorm_bwd, *ctx.saved_tensors, ctx.scale, ctx.needs_input_grad[:3], dtotal, dy)
    return (*grads, None, None)


add_rmsnorm.register_autograd(_add_rmsnorm_backward, setup_context=_add_rmsnorm_setup)


class _AddRmsNorm(torch.autograd.Function):
    """add_rmsnorm under eager autograd, without the dispatcher's host time."""

    @staticmethod
    def forward(ctx, x, residual, weight, scale, eps):
        total, y, rstd = _add_rmsnorm_eager(x, residual, weight, scale, eps)
        ctx.scale = scale
        ctx.save_for_backward(total, weight, rstd)
        ctx.set_materialize_grads(False)
        return total, y

    @staticmethod
    def _grads(ctx, dtotal, dy):
        grads = _add_rmsnorm_grads(_add_rmsnorm_bwd_eager, *ctx.saved_tensors, ctx.scale, ctx.needs_input_grad[:3], dtotal, dy)
        return (*grads, None, None)

    _once = staticmethod(torch.autograd.function.once_differentiable(_grads.__func__))

    @staticmethod
    def backward(ctx, dtotal, dy):
        # the wrapper is for a caller that records the backward; without one it is time alone
        return (_AddRmsNorm._once if _is_grad_enabled() else _AddRmsNorm._grads)(ctx, dtotal, dy)


def _add_rmsnorm_mx_eager(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor, scale: float,
                          eps: float, fmt: str) -> tuple[Optional[torch.Tensor], torch.Tensor, torch.Tensor]:
    """m3_add_rmsnorm_mx over the last dimension: (total, or None without a residual; data, scales)."""
    _native.require_gpu(x, residual, weight)
    with on_device(x):
        x2 = _rows_of(x)
        total = None if residual is None else torch.empty_like(x2)
        rows, d = x2.shape
        data, scales = _mx_empty(rows, d, fmt, x2)
        if rows:
            _native.add_rmsnorm_mx(x2, None if residual is None else _rows_of(residual), weight.contiguous(), scale, eps,
                                   total, fmt, data, scales)
    return total if total is None or x2 is x else total.view(x.shape), data, scales


@torch.library.custom_op(f"{NS}::add_rmsnorm_mx", mutates_args=())
def add_rmsnorm_mx(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor, scale: float, eps: float,
                   fmt: str) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """_add_rmsnorm_mx_eager as an op; the first output is empty without a residual."""
    total, data, scales = _add_rmsnorm_mx_eager(x, residual, weight, scale, eps, fmt)
    return x.new_empty(0) if total is None else total, data, scales


@add_rmsnorm_mx.register_fake
def _(x, residual, weight, scale, eps, fmt):
    return (x.new_empty((0,) if residual is None else x.shape), *_mx_empty(x.numel() // x.shape[-1], x.shape[-1], fmt, x))


def _mx_linear_eager(x_data: torch.Tensor, x_scales: torch.Tensor, x_format: str, w_data: torch.Tensor,
                     w_scales: torch.Tensor, k: int, residual: Optional[torch.Tensor], scale: float,
                     dtype: torch.dtype) -> torch.Tensor:
    """m3_mx_linear: (rows, n) in `dtype`, the residual's where one is given."""
    _native.require_gpu(x_data, x_scales, w_data, w_scales, residual)
    with on_device(x_data):
        rows, n = x_data.shape[0], w_data.shape[0]
        out = x_data.new_empty((rows, n), dtype=dtype)
        if rows and n:
            _native.mx_linear(x_data, x_scales, x_format, w_data, w_scales, k,
                              None if residual is None else _rows_of(residual), scale, out)
    return out


mx_linear = torch.library.custom_op(f"{NS}::mx_linear", _mx_linear_eager, mutates_args=())


@mx_linear.register_fake
def _(x_data, x_scales, x_format, w_data, w_scales, k, residual, scale, dtype):
    return x_data.new_empty((x_data.shape[0], w_data.shape[0]), dtype=dtype)


@functools.lru_cache(maxsize=1024)
def _takes_tensor(rows: int, n: int, k: int, x_dtype: torch.dtype, dtype: torch.dtype, before: int) -> bool:
    return _native.mx_linear_takes_tensor(rows, n, k, x_dtype, dtype, before)


def mx_linear_takes_tensor(x: torch.Tensor, n: int, k: int, dtype: torch.dtype, before: int) -> bool:
    """True where one launch quantises x, behind its norm or gate, and multiplies (sizes and types alone decide; under
    torch.compile sizes may be symbolic, and two launches run)."""
    return not _is_compiling() and x.numel() > 0 and _takes_tensor(x.numel() // x.shape[-1], n, k, x.dtype, dtype, before)


def _mx_linear_tensor_eager(x: torch.Tensor, norm_weight: Optional[torch.Tensor], eps: float, gated: bool, w_data: torch.Tensor,
                            w_scales: torch.Tensor, residual: Optional[torch.Tensor], scale: float, dtype: torch.dtype) -> torch.Tensor:
    """m3_mx_linear_tensor: (rows, n) in `dtype`."""
    _native.require_gpu(x, norm_weight, w_data, w_scales, residual)
    with on_device(x):
        x2 = _rows_of(x)
        out = x2.new_empty((x2.shape[0], w_data.shape[0]), dtype=dtype)
        _native.mx_linear_tensor(x2, None if norm_weight is None else norm_weight.contiguous(), eps, gated, w_data, w_scales,
                                 None if residual is None else _rows_of(residual), scale, out)
    return out


mx_linear_tensor = torch.library.custom_op(f"{NS}::mx_linear_tensor", _mx_linear_tensor_eager, mutates_args=())


@mx_linear_tensor.register_fake
def _(x, norm_weight, eps, gated, w_data, w_scales, residual, scale, dtype):
    return x.new_empty((x.numel() // x.shape[-1], w_data.shape[0]), dtype=dtype)


def _sample_tokens_eager(logits: torch.Tensor, u: torch.Tensor, temperatures: Optional[torch.Tensor], temperature: float,
                         top_ks: Optional[torch.Tensor], top_k: int, top_ps: Optional[torch.Tensor], top_p: float,
                         min_ps: Optional[torch.Tensor], min_p: float, logprob: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """m3_sample_tokens on logits (rows, vocab): (tokens (rows,) int64, log probabilities (rows,), empty unless asked
    for). A setting is the tensor (rows,), or where that is None the number."""
    _native.require_gpu(logits, u, temperatures, top_ks, top_ps, min_ps)
    with on_device(logits):
        rows = logits.shape[0]
        token = logits.new_empty(rows, dtype=torch.int64)
        lp = logits.new_empty(rows if logprob else 0, dtype=torch.float32)
        each = [n if t is None else t.contiguous()
                for t, n in ((temperatures, temperature), (top_ks, top_k), (top_ps, top_p), (min_ps, min_p))]
        if rows:
            _native.sample_tokens(_rows_of(logits), u.contiguous(), *each, token, lp if logprob else None)
    return token, lp


sample_tokens = torch.library.custom_op(f"{NS}::sample_tokens", _sample_tokens_eager, mutates_args=())


@sample_tokens.register_fake
def _(logits, u, temperatures, temperature, top_ks, top_k, top_ps, top_p, min_ps, min_p, logprob):
    rows = logits.shape[0]
    return logits.new_empty(rows, dtype=torch.int64), logits.new_empty(rows if logprob else 0, dtype=torch.float32)


def mx_quantize_fast(x, fmt, gated):
    return (_mx_quantize_eager if _plain(x) else mx_quantize)(x, fmt, gated)


def mx_dequantize_fast(data, scales, fmt, k, dtype):
    return (_mx_dequantize_eager if _plain(data, scales) else mx_dequantize)(data, scales, fmt, k, dtype)


def add_rmsnorm_fast(x, residual, weight, scale, eps):
    if not _plain(x, residual, weight):
        return add_rmsnorm(x, residual, weight, scale, eps)[:2]
    if _is_grad_enabled() and (x.requires_grad or residual.requires_grad or weight.requires_grad):
        return _AddRmsNorm.apply(x, residual, weight, scale, eps)
    return _add_rmsnorm_eager(x, residual, weight, scale, eps, False)[:2]


def add_rmsnorm_mx_fast(x, residual, weight, scale, eps, fmt):
    return (_add_rmsnorm_mx_eager if _plain(x, residual, weight) else add_rmsnorm_mx)(x, residual, weight, scale, eps, fmt)


def mx_linear_fast(x_data, x_scales, x_format, w_data, w_scales, k, residual, scale, dtype):
    fn = _mx_linear_eager if _plain(x_data, x_scales, w_data, w_scales, residual) else mx_linear
    return fn(x_data, x_scales, x_format, w_data, w_scales, k, residual, scale, dtype)


def mx_linear_tensor_fast(x, norm_weight, eps, gated, w_data, w_scales, residual, scale, dtype):
    fn = _mx_linear_tensor_eager if _plain(x, norm_weight, w_data, w_scales, residual) else mx_linear_tensor
    return fn(x, norm_weight, eps, gated, w_data, w_scales, residual, scale, dtype)


def sample_tokens_fast(logits, u, temperatures, temperature, top_ks, top_k, top_ps, top_p, min_ps, min_p, logprob):
    fn = _sample_tokens_eager if _plain(logits, u, temperatures, top_ks, top_ps, min_ps) else sample_tokens
    return fn(logits, u, temperatures, temperature, top_ks, top_k, top_ps, top_p, min_ps, min_p, logprob)
