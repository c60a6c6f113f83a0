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
    # A model has hundreds of small gradients: each of these passes over them is one C call per tensor.
    grads = [g for g in [p.grad for p in params] if g is not None]
    if len(set(map(id, grads))) < len(grads):
        grads = list({id(g): g for g in grads}.values())
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
    for layout in {g.layout for g in grads}:
        if layout is not torch.strided:
            raise TypeError(f"clip_grad_norm_ takes dense gradients, got {layout}")
    dtypes = [g.dtype for g in grads]
    codes = {d: _native.dtype_code(d) for d in set(dtypes)}
    _native.require_gpu(grads[0])
    if len(set(map(torch.Tensor.get_device, grads))) > 1:
        raise ValueError(f"gradients must be on one GPU, got {sorted({str(g.device) for g in grads})}")
    whole = grads  # what the kernels work on: the gradients themselves or contiguous copies
    if not all(map(torch.Tensor.is_contiguous, grads)):
        for g in grads:
            if not g.is_contiguous() and any(n > 1 and s == 0 for n, s in zip(g.shape, g.stride())):
                raise ValueError("a gradient whose elements share memory (expanded) cannot be clipped in place")
        whole = [g.detach().contiguous() for g in grads]
    args = (list(map(torch.Tensor.data_ptr, whole)), list(map(torch.Tensor.numel, whole)),
            [codes[d] for d in dtypes], kind)
    with ops.on_device(grads[0]):
        norm = torch.empty((), dtype=torch.float32, device=grads[0].device)
        if error_if_nonfinite:
            _native.clip_grad_norm(*args, None, norm)
            if not math.isfinite(norm.item()):
                raise RuntimeError(f"the norm of the gradients is {norm.item()}: they were not clipped")
        _native.clip_grad_norm(*args, max_norm, norm)
        torch.autograd.graph.increment_version(grads)
        if whole is not grads:
            with torch.no_grad():
                for g, t in zip(grads, whole):
                    if t.data_ptr() != g.data_ptr():
                        g.copy_(t)
    return norm
