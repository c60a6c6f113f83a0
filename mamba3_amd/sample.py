"""The next token of each row of logits from given random numbers, on the HIP kernels behind `m3_sample_tokens`
(mamba3/block.py:208-222 draws with torch.multinomial from the whole softmax).
"""

from __future__ import annotations

import math

import torch

from . import _native, ops
from .mx import refuse_gradients


def _setting(name: str, v, least: float, most: float, shape, device, dtype) -> tuple[torch.Tensor | None, float]:
    """A setting as (tensor by row, number)."""
    if isinstance(v, torch.Tensor):
        if v.shape != shape or v.device != device:
            raise ValueError(f"{name} has shape {tuple(v.shape)} on {v.device}, expected {tuple(shape)} on {device}")
        if dtype == torch.int32 and v.dtype == torch.int64:
            v = v.clamp(-1, 2**31 - 1).to(torch.int32)
        if v.dtype != dtype:
            raise TypeError(f"{name} by row must be {dtype}, got {v.dtype}")
        return v.reshape(-1), 0
    v = int(v) if dtype is torch.int32 else float(v)
    if not least <= v <= most:
        raise ValueError(f"{name} must lie in [{least}, {most}], got {v}")
    return None, v


def sample_tokens(logits: torch.Tensor, u: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
                  return_logprob: bool = False):
    """Tokens (...) int64 for logits (..., vocab), fp32 or bf16, from u (...) fp32 in [0, 1), one random number
    each. Each setting is a number or a tensor (...) with one for each row (fp32; top_k int32 or int64).

    Tokens are ordered by logit, equal ones by index. With masses exp((z - max z) / temperature), kept are the
    first `top_k` (0: all); of these the shortest run from the first on whose mass reaches `top_p` of theirs (1: all,
    0: the first); of these the ones with at least `min_p` of the first's mass. The answer is the first kept token
    whose running mass, in that order, passes u times the kept mass: a smaller u gives a likelier token. A temperature
    of 0 takes the first. With `return_logprob` the result is (tokens, the logs of their shares of the kept mass).

    NaN logits count as -inf, which is never chosen; a row with nothing else gives -1. Settings by row are not checked on
    the host: a temperature below 0 or NaN acts as 0, top_k below 1 as all, top_p and min_p as their nearest end, NaN as
    not given. The same inputs give the same tokens: sums do not depend on their order. vocab is at most 2^22."""
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"sample_tokens needs logits (..., vocab), got shape {tuple(logits.shape)}")
    shape = logits.shape[:-1]
    _native.dtype_code(logits.dtype)
    if u.shape != shape or u.device != logits.device:
        raise ValueError(f"u has shape {tuple(u.shape)} on {u.device}, expected {tuple(shape)} on {logits.device}")
    if u.dtype != torch.float32:
        raise TypeError(f"u must be float32, got {u.dtype}")
    if logits.shape[-1] > 1 << 22:
        raise ValueError(f"sample_tokens takes at most {1 << 22} tokens, got {logits.shape[-1]}")
    if return_logprob:
        refuse_gradients("sample_tokens", logits)
    args = []
    for name, v, most, dtype in (("temperature", temperature, math.inf, torch.float32), ("top_k", top_k, 2**62, torch.int32),
                                 ("top_p", top_p, 1.0, torch.float32), ("min_p", min_p, 1.0, torch.float32)):
        args += _setting(name, v, 0, most, shape, logits.device, dtype)
    _native.require_gpu(logits)
    z = logits.detach() if logits.requires_grad else logits
    if len(shape) == 1:
        got = ops.sample_tokens_fast(z, u, *args, return_logprob)
        return got if return_logprob else got[0]
    token, lp = ops.sample_tokens_fast(z.reshape(-1, z.shape[-1]), u.reshape(-1), *args, return_logprob)
    return (token.view(shape), lp.view(shape)) if return_logprob else token.view(shape)
