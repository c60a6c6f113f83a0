"""The language model's loss without its logits.

    z = hidden weight^T,   loss = log sum_v exp z_v - z_target

(mamba3/block.py:183-192 keeps the (rows, vocab) logits and several copies of them), on the HIP
kernels behind `m3_linear_xent_fwd` / `m3_linear_xent_bwd` (the `mamba3_amd::linear_xent` op): the
forward leaves one number per row, the backward works through the vocabulary in pieces.
"""

from __future__ import annotations

import torch

from . import _native, ops


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, target: torch.Tensor,
                         ignore_index: int = -100, reduction: str = "mean") -> torch.Tensor:
    """Cross entropy of softmax(hidden weight^T) against target: hidden (..., d_model) and weight
    (vocab, d_model), both fp32 or both bf16, target (...) int64, on one GPU. Returns an fp32 scalar
    ("mean" over the rows that count, NaN where none does, or "sum") or a loss per row ("none").
    Differentiable in hidden and weight; sums are fp32 and run in a fixed order. Under bf16 autocast both
    are taken in bf16.

    A row whose target is `ignore_index` counts nowhere: its loss and its gradients are zero whatever
    `hidden` holds there. Any other target outside [0, vocab) is not checked on the host: it makes the
    row's loss, and the gradients that it enters, NaN."""
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"hidden {tuple(hidden.shape)} and weight {tuple(weight.shape)} do not fit "
                         "(..., d_model) and (vocab, d_model)")
    if target.shape != hidden.shape[:-1]:
        raise ValueError(f"target has shape {tuple(target.shape)}, expected {tuple(hidden.shape[:-1])}")
    if target.dtype != torch.int64:
        raise TypeError(f"target must be int64, got {target.dtype}")
    if reduction not in _native.REDUCTIONS:
        raise ValueError(f"reduction must be 'none', 'mean' or 'sum', got {reduction!r}")
    if weight.numel() == 0:
        raise ValueError("linear_cross_entropy needs a vocabulary and d_model of at least 1")
    hidden, weight = ops.autocast(hidden, weight)
    ops.check_alike("linear_cross_entropy", hidden, weight)
    if target.device != hidden.device:
        raise ValueError(f"target is on {target.device}, hidden on {hidden.device}")
    if target.numel() == 0:
        # no rows: every gradient is zero, and the graph still reaches both inputs
        none = (hidden.reshape(-1, hidden.shape[-1]) @ weight.t()).float().sum(-1).reshape(target.shape)
        return none if reduction == "none" else none.sum() if reduction == "sum" else none.mean()
    return ops.linear_xent_fast(hidden, weight, target, int(ignore_index), _native.REDUCTIONS[reduction])
