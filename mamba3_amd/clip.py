"""Clipping of gradients by their global norm, on the HIP kernels behind `m3_clip_grad_norm`."""

from __future__ import annotations

import math
from typing import Iterable

import torch

from . import _native, ops


def _reaches(terms: list[tuple[int, int, int]], target: int, budget: list[int]) -> bool:
    """Whether target = sum of c x over the terms (c, lo, hi), by falling c > 0, for whole x in [lo, hi]."""
    if not terms:
        return target == 0
    (c, lo, hi), rest = terms[0], terms[1:]
    least, most = sum(k * a for k, a, _ in rest), sum(k * b for k, _, b in rest)
    lo, hi = max(lo, -((most - target) // c)), min(hi, (target - least) // c)
    step = math.gcd(*[k for k, _, _ in rest])  # what the rest comes in
    if step == 0:
        return lo <= hi and target == c * lo
    common = math.gcd(c, step)
    if target % common:
        return False
    m = step // common
    first = (target // common) * pow(c // common, -1, m) % m  # of the x that leave a multiple of step
    for x in range(lo + (first - lo) % m, hi + 1, m):
        budget[0] -= 1
        if budget[0] < 0:
            raise ValueError("strided gradients that lie within one another and could not be told apart")
        if _reaches(rest, target - c * x, budget):
            return True
    return False


def _terms(strides: list[tuple[int, int, int]]) -> list[tuple[int, int, int]]:
    """(c, lo, hi) with equal c joined, by falling c."""
    joined: dict[int, tuple[int, int]] = {}
    for c, lo, hi in strides:
        a, b = joined.get(c, (0, 0))
        joined[c] = (a + lo, b + hi)
    return sorted(((c, *r) for c, r in joined.items()), reverse=True)


def _refuse_shared_memory(grads: list[torch.Tensor]) -> None:
    """Raises where an element of a strided gradient is one of another gradient, or twice its own."""
    def dims_of(g):
        return sorted(((s * g.element_size(), n) for n, s in zip(g.shape, g.stride()) if n > 1), reverse=True)

    spans = []
    for g in grads:
        at, size = g.data_ptr(), g.element_size()
        if g.numel() == 0:
            continue
        if g.is_contiguous():
            spans.append((at, at + g.numel() * size, True, g))
            continue
        dims = dims_of(g)
        if dims[-1][0] == 0:
            raise ValueError("a gradient whose elements share memory (expanded) cannot be clipped in place")
        # two places that differ first in dimension k, and are the same
        for k, (s, n) in enumerate(dims):
            below = sum((m - 1) * t for t, m in dims[k + 1:])
            later = _terms([(t, 1 - m, m - 1) for t, m in dims[k + 1:]])
            if any(_reaches(later, off - s * x, [1 << 16]) for x in range(1, min(n - 1, (below + size - 1) // s) + 1)
                   for off in range(1 - size, size)):
                raise ValueError("a gradient whose elements share memory cannot be clipped in place")
        spans.append((at, at + size + sum((n - 1) * s for s, n in dims), False, g))
    spans.sort(key=lambda v: v[0])
    for i, (at, end, whole, g) in enumerate(spans):
        for at2, _, whole2, g2 in spans[i + 1:]:
            if at2 >= end:
                break
            if whole and whole2:
                continue  # the kernels' own check finds these
            # a place of the first minus a place of the second is less than an element apart
            terms = _terms([(s, 0, n - 1) for s, n in dims_of(g)] + [(s, 1 - n, 0) for s, n in dims_of(g2)])
            size, size2 = g.element_size(), g2.element_size()
            unit = math.gcd(at2 - at, size, size2, *[c for c, _, _ in terms])  # what all places are apart by
            if any(_reaches(terms, at2 - at + off, [1 << 16]) for off in range(unit - size, size2, unit)):
                raise ValueError("gradients that overlap in memory cannot be clipped in place")


def clip_grad_norm_(parameters: torch.Tensor | Iterable[torch.Tensor], max_norm: float,
                    norm_type: float = 2.0, error_if_nonfinite: bool = False) -> torch.Tensor:
    """Scales the gradients of `parameters` in place by min(1, max_norm / (norm + 1e-6)) and returns
    norm, the norm of all their elements together before that (an fp32 scalar on their GPU): the
    2-norm, or for norm_type inf the largest absolute value. Gradients are fp32 or bf16, in any
    mixture, on one GPU; parameters without one are left out, one that is listed twice counts
    once, and gradients that share memory otherwise are refused. Nothing waits for the GPU, unless
    error_if_nonfinite asks to raise, before anything is scaled, where the norm is NaN or infinite;
    otherwise such a norm scales by NaN or 0."""
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
        _refuse_shared_memory(grads)
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
