"""The gated MLP of a residual block as one differentiable operator.

    y = [residual +] scale * (silu(x w_gate^T) * (x w_up^T)) w_down^T

(mamba3/block.py:16-26 with the residual add of block.py:86-91), on the HIP kernels behind
`m3_swiglu_mlp_fwd` / `m3_swiglu_mlp_bwd` (the `mamba3_amd::swiglu_mlp` op): both projections, the
activation and the product are one kernel, the down projection adds the residual, and no
intermediate but the hidden activations and, for the backward, the gate and up values is stored.
"""

from __future__ import annotations

import torch

from . import _native, ops


def swiglu_mlp(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
               residual: torch.Tensor | None = None, scale: float = 1.0) -> torch.Tensor:
    """x (..., d_model), w_gate and w_up (d_ff, d_model), w_down (d_model, d_ff), residual of x's
    shape; all fp32 or all bf16, on one GPU. Returns x's shape and dtype. Differentiable in every
    tensor; sums are fp32 and run in a fixed order. Under bf16 autocast the products run in bf16 and the
    residual is added in its own type. Without gradients, at most 8 bf16 rows run on the decode kernels (`m3_small_swiglu`, `m3_small_linear`) where they take the shape."""
    if x.dim() < 1 or w_gate.dim() != 2 or w_up.dim() != 2 or w_down.dim() != 2:
        raise ValueError("swiglu_mlp expects x (..., d_model) and two-dimensional weights")
    ff, d = w_gate.shape
    if x.shape[-1] != d or tuple(w_up.shape) != (ff, d) or tuple(w_down.shape) != (d, ff):
        raise ValueError(f"x {tuple(x.shape)}, w_gate {tuple(w_gate.shape)}, w_up {tuple(w_up.shape)} and "
                         f"w_down {tuple(w_down.shape)} do not fit (..., d), (f, d), (f, d), (d, f)")
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"residual has shape {tuple(residual.shape)}, expected {tuple(x.shape)}")
    x, w_gate, w_up, w_down = ops.autocast(x, w_gate, w_up, w_down)
    if residual is not None and residual.dtype != x.dtype and torch.is_autocast_enabled("cuda"):
        # the residual stream keeps its type
        return residual + swiglu_mlp(x, w_gate, w_up, w_down, None, scale)
    ins = (x, w_gate, w_up, w_down) if residual is None else (x, w_gate, w_up, w_down, residual)
    ops.check_alike("swiglu_mlp", *ins)
    if d == 0 or ff == 0:
        raise ValueError("swiglu_mlp needs d_model and d_ff of at least 1")
    scale = float(scale)
    if x.numel() == 0:
        # no rows: every gradient is zero, and the graph still reaches each input
        out = x.reshape(-1, d) @ w_gate.t() * (x.reshape(-1, d) @ w_up.t()) @ w_down.t()
        return (out.reshape(x.shape) if residual is None else residual + out.reshape(x.shape))
    keep = torch.is_grad_enabled() and any(t.requires_grad for t in ins)
    if not keep and (residual is not None or scale == 1.0) and x.is_contiguous():
        x2 = x.reshape(-1, d)
        if (ops.small_proj_usable(x2, w_gate, w_up, w_down) and _native.small_proj_ok(x2.shape[0], ff)
                and (residual is None or residual.is_contiguous())):
            with ops.on_device(x):
                h = ops.small_swiglu_fast(x2, None, 0.0, w_gate, w_up)
                res = None if residual is None else residual.reshape(-1, d)
                return ops.small_linear_fast(h, None, 0.0, w_down, res, scale).view(x.shape)
    return ops.swiglu_mlp_fast(x, w_gate, w_up, w_down, residual, scale, keep)
