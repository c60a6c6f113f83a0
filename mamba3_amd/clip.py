"""Clipping of gradients by their global norm, on the HIP kernels behind `m3_clip_grad_norm`."""

from __future__ import annotations

import math
from typing import Iterable

import torch

from . import _native, ops


def clip_grad_norm_(parameters: torch.Tensor | Iterable[torch.Tensor], max_norm: float,
                    norm_type: float = 2.0, error_if_nonfinite: bool = False) -> torch.Tensor:
    """Scales the gradients of `parameters` in place by min(1, max_norm / (norm + 1e-6)) and returns
    norm, the norm of all their elements together before that (an fp32 scalar on their GPU): the
    2-norm, or for norm_type inf the largest absolute value. Gradients are fp32 or bf16, in any
    mixture, on one GPU; parameters without one are left out, and one that is listed twice counts
    once. Nothing waits for the GPU, unless error_if_nonfinite asks to raise, before anything is
    scaled, where the norm is NaN or infinite; otherwise such a norm scales by NaN or 0."""
    params = (parameters,) if isinstance(parameters, torch.Tensor) else parameters
    # the same gradient listed twice counts once
    grads = list({id(g): g for g in [p.grad for p in params] if g is not None}.values())
    max_norm, norm_type = float(max_norm), float(norm_type)
    if norm_type == 2.0:
        kind = _native.NORM_L2
    elif norm_type == math.inf:
        kind = _native.NORM_MAX
    else:
        raise ValueError(f"norm_type must be 2 or inf, got {norm_type}")
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    if not grads:
        return torch.tensor(0.0)
    device = grads[0].device
    for g in grads:
        if g.layout is not torch.strided:
            raise TypeError(f"clip_grad_norm_ takes dense gradients, got {g.layout}")
        if g.device != device:
            raise ValueError(f"gradients must be on one GPU, got {device} and {g.device}")
    codes = [_native.dtype_code(g.dtype) for g in grads]
    _native.require_gpu(grads[0])
    whole = grads  # what the kernels work on: the gradients themselves or contiguous copies
    strided = [g for g in grads if not g.is_contiguous()]
    if strided:
        for g in strided:
            if any(n > 1 and s == 0 for n, s in zip(g.shape, g.stride())):
                raise ValueError("a gradient whose elements share memory (expanded) cannot be clipped in place")
        whole = [g.detach().contiguous() for g in grads]
    ptrs, sizes = [t.data_ptr() for t in whole], [t.numel() for t in whole]
    end = 0
    for at, n, code in sorted(zip(ptrs, sizes, codes)):
        if n:
            if at < end:
                raise ValueError("gradients that overlap in memory cannot be clipped in place")
            end = at + n * (2 if code == _native.M3_DTYPE_BF16 else 4)
    with ops.on_device(grads[0]):
        norm = torch.empty((), dtype=torch.float32, device=device)
        if error_if_nonfinite:
            _native.clip_grad_norm(ptrs, sizes, codes, kind, None, norm)
            if not math.isfinite(norm.item()):
                raise RuntimeError(f"the norm of the gradients is {norm.item()}: they were not clipped")
        _native.clip_grad_norm(ptrs, sizes, codes, kind, max_norm, norm)
        torch.autograd.graph.increment_version(grads)
        if strided:
            with torch.no_grad():
                for g, t in zip(grads, whole):
                    if t.data_ptr() != g.data_ptr():
                        g.copy_(t)
    return norm
