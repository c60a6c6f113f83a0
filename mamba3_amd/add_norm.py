"""The residual's addition with the norm behind it as one operator.

    total = residual + scale * x,    y = total / sqrt(mean total^2 + eps) * weight

(mamba3/block.py:84-91 with the RMSNorm of mamba3/mamba3.py:19-35), on the HIP kernels behind
`m3_add_rmsnorm_fwd` / `m3_add_rmsnorm_bwd` and `m3_add_rmsnorm_mx`. The norm is of the sum as it is stored; y
is computed in fp32 and rounded once, where RMSNorm rounds 1 / sqrt and its product with x on the way.
"""

from __future__ import annotations

import torch

from . import ops
from .mx import MXTensor, _mx, check_format, refuse_gradients


def _check(what: str, x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor) -> None:
    if x.dim() < 1 or weight.dim() != 1 or x.shape[-1] != weight.shape[0] or weight.shape[0] < 1:
        raise ValueError(f"x {tuple(x.shape)} and weight {tuple(weight.shape)} do not fit (..., d) and (d,)")
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"residual has shape {tuple(residual.shape)}, expected {tuple(x.shape)}")
    ops.check_alike(what, x, weight) if residual is None else ops.check_alike(what, x, residual, weight)


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, scale: float = 1.0,
                 eps: float = 1e-5) -> tuple[torch.Tensor, torch.Tensor]:
    """(total, y) for x and residual (..., d) and weight (d,), all fp32 or all bf16, on one GPU. Differentiable in
    the three tensors through both results; sums run in a fixed order."""
    _check("add_rms_norm", x, residual, weight)
    scale, eps = float(scale), float(eps)
    if x.numel() == 0:
        # no rows: every gradient is zero, and the graph still reaches each input
        total = residual + scale * x
        return total, total * weight
    return ops.add_rmsnorm_fast(x, residual, weight, scale, eps)


def add_rms_norm_mx(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, scale: float = 1.0,
                    eps: float = 1e-5, format: str = "e4m3") -> tuple[torch.Tensor, MXTensor]:
    """add_rms_norm with y as microscaled values, for the product that reads it. Without a residual total is x (and
    scale is not used). No backward."""
    check_format(format)
    refuse_gradients("add_rms_norm_mx", x, residual, weight)
    _check("add_rms_norm_mx", x, residual, weight)
    total, data, scales = ops.add_rmsnorm_mx_fast(x, residual, weight, float(scale), float(eps), format)
    return (x if residual is None else total), _mx(data, scales, x.shape, format)
