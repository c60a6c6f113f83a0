"""Microscaled values: blocks of 32 along the last dimension share a power of two, elements have 4 bits (e2m1)
or 8 (e4m3). Quantisation, and products of such activations with 4-bit weights, on the HIP kernels behind
`m3_mx_quantize`, `m3_mx_dequantize` and `m3_mx_linear`.

A block's power of two is the smallest under which its largest magnitude rounds to an element, so nothing
saturates; elements round to nearest, ties to even. A block that holds an infinity or NaN is NaN.
"""

from __future__ import annotations

import math

import torch

from . import _native, ops


def check_format(fmt: str) -> None:
    if fmt not in _native.MX_FORMATS:
        raise ValueError(f"format must be 'e2m1' or 'e4m3', got {fmt!r}")


def refuse_gradients(what: str, *tensors: torch.Tensor | None) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{what} has no backward: call it under torch.no_grad(), or detach its inputs")


class MXTensor:
    """Microscaled values of `shape`, as two uint8 tensors with a row for each row of the last dimension: `data`
    (rows, kp) for e4m3 or (rows, kp / 2) for e2m1 (the even index in a byte's low half), where kp is
    shape[-1] rounded up to 128, and `scales` (rows, kp / 32), exponents + 127 (255: NaN). What lies behind
    shape[-1] is zeros."""

    __slots__ = ("data", "scales", "shape", "format")

    def __init__(self, data: torch.Tensor, scales: torch.Tensor, shape, format: str):
        check_format(format)
        shape = torch.Size(shape)
        if len(shape) < 1 or shape[-1] < 1:
            raise ValueError(f"MXTensor needs a last dimension of at least 1, got shape {tuple(shape)}")
        k = shape[-1]
        rows, kp = shape[0] if len(shape) == 2 else math.prod(shape[:-1]), _native.mx_padded(k)
        if data.shape != (rows, kp if format == "e4m3" else kp // 2) or scales.shape != (rows, kp // 32):
            raise ValueError(f"data and scales must have shapes {(rows, _native.mx_row_bytes(k, format))} and {(rows, kp // 32)}, got {tuple(data.shape)} "
                             f"and {tuple(scales.shape)}")
        for name, t in (("data", data), ("scales", scales)):
            if t.dtype is not torch.uint8 or not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous uint8, got {t.dtype} with strides {t.stride()}")
        if data.device != scales.device:
            raise ValueError(f"data is on {data.device}, scales on {scales.device}")
        if data.is_cuda and not torch.compiler.is_compiling() and (data.data_ptr() % 16 or scales.data_ptr() % 4):
            raise ValueError("data must be 16-byte aligned and scales 4-byte aligned")
        self.data, self.scales, self.shape, self.format = data, scales, shape, format

    @property
    def device(self) -> torch.device:
        return self.data.device

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The values, in fp32 or bf16 (both hold them exactly, but for results below 2^-126 and past the largest number)."""
        _native.dtype_code(dtype)
        out = ops.mx_dequantize_fast(self.data, self.scales, self.format, self.shape[-1], dtype)
        return out if len(self.shape) == 2 else out.view(self.shape)

    def __repr__(self) -> str:
        return f"MXTensor(shape={tuple(self.shape)}, format={self.format!r}, device={str(self.device)!r})"


def _mx(data: torch.Tensor, scales: torch.Tensor, shape, format: str) -> MXTensor:
    """An MXTensor of what the kernels wrote."""
    t = MXTensor.__new__(MXTensor)
    t.data, t.scales, t.shape, t.format = data, scales, shape if type(shape) is torch.Size else torch.Size(shape), format
    return t


def quantize_mx(x: torch.Tensor, format: str = "e2m1") -> MXTensor:
    """x (..., k), fp32 or bf16 on a GPU, as microscaled values. No backward."""
    check_format(format)
    shape = x.shape
    if len(shape) < 1 or shape[-1] < 1:
        raise ValueError(f"quantize_mx needs a last dimension of at least 1, got shape {tuple(shape)}")
    _native.dtype_code(x.dtype)
    refuse_gradients("quantize_mx", x)
    return _mx(*ops.mx_quantize_fast(x, format, False), shape, format)


def silu_mul_mx(gate_up: torch.Tensor, format: str = "e4m3") -> MXTensor:
    """silu(gate) * up as microscaled values, from gate_up (..., 2 k) that holds the gate in its first half
    (mamba3/block.py:16-26 between its products), rounded as the exact product would be. No backward."""
    check_format(format)
    if gate_up.dim() < 1 or gate_up.shape[-1] < 2 or gate_up.shape[-1] % 2:
        raise ValueError(f"silu_mul_mx needs an even last dimension of at least 2, got shape {tuple(gate_up.shape)}")
    _native.dtype_code(gate_up.dtype)
    refuse_gradients("silu_mul_mx", gate_up)
    return _mx(*ops.mx_quantize_fast(gate_up, format, True), (*gate_up.shape[:-1], gate_up.shape[-1] // 2), format)


def mx_linear(x: MXTensor | torch.Tensor, weight: MXTensor, residual: torch.Tensor | None = None, scale: float = 1.0,
              out_dtype: torch.dtype | None = None, norm_weight: torch.Tensor | None = None, eps: float = 1e-5,
              gated: bool = False) -> torch.Tensor:
    """[residual +] scale * x weight^T for weight (n, k) in e2m1 and x (..., k): microscaled in either format, or
    a tensor, which is quantised to e4m3 on the way. The result (..., n) has out_dtype: by default the residual's type,
    x's, or bf16. No backward.

    A tensor is first normed where norm_weight (k,) is given (add_rms_norm_mx with eps and without a residual), or with `gated`
    is (..., 2 k) and enters as silu_mul_mx gives it. The results are those of the separate calls; for few rows one launch does it.

    Sums are fp32. For a bf16 result the matrix instructions align the 128 products that they add at a time at about
    2^-13 of the largest where x is e4m3; an fp32 result has no such step."""
    if not isinstance(weight, MXTensor) or weight.format != "e2m1" or len(weight.shape) != 2:
        raise ValueError("mx_linear needs a two-dimensional e2m1 MXTensor as weight")
    n, k = weight.shape
    plain, given = not isinstance(x, MXTensor), x.shape
    if plain:
        if len(given) < 1:
            raise ValueError("mx_linear expects x (..., k)")
        refuse_gradients("mx_linear", x)
        _native.dtype_code(x.dtype)
    elif gated or norm_weight is not None:
        raise ValueError("norm_weight and gated are for a tensor, x is microscaled already")
    if given[-1] != (2 * k if gated else k) or n < 1:
        raise ValueError(f"x {tuple(given)} and weight {tuple(weight.shape)} do not fit (..., {'2 k' if gated else 'k'}) and (n, k)")
    if norm_weight is not None:
        if gated:
            raise ValueError("either norm_weight or gated")
        if norm_weight.shape != (k,) or norm_weight.dtype != x.dtype or norm_weight.device != x.device:
            raise ValueError(f"norm_weight must be {x.dtype} of shape {(k,)} on {x.device}, got {norm_weight.dtype} "
                             f"{tuple(norm_weight.shape)} on {norm_weight.device}")
        refuse_gradients("mx_linear", norm_weight)
    if out_dtype is None:
        out_dtype = residual.dtype if residual is not None else x.dtype if plain else torch.bfloat16
    _native.dtype_code(out_dtype)
    at = weight.data.device
    if (x if plain else x.data).device != at:
        # a tensor on the host is refused for what it is
        _native.require_gpu(x if plain else x.data)
        raise ValueError(f"x is on {x.device}, weight on {at}")
    shape = (given[0], n) if len(given) == 2 else (*given[:-1], n)
    if residual is not None:
        if residual.shape != shape or residual.dtype != out_dtype or residual.device != at:
            raise ValueError(f"residual must be {out_dtype} of shape {shape} on {x.device}, got {residual.dtype} "
                             f"{tuple(residual.shape)} on {residual.device}")
        refuse_gradients("mx_linear", residual)
    before = _native.MX_GATED if gated else _native.MX_AS_IS if norm_weight is None else _native.MX_NORMED
    if plain and ops.mx_linear_takes_tensor(x, n, k, out_dtype, before):
        out = ops.mx_linear_tensor_fast(x, norm_weight, float(eps), gated, weight.data, weight.scales, residual, float(scale), out_dtype)
    else:
        q = x
        if gated:
            q = silu_mul_mx(x)
        elif norm_weight is not None:
            q = _mx(*ops.add_rmsnorm_mx_fast(x, None, norm_weight, 1.0, float(eps), "e4m3")[1:], x.shape, "e4m3")
        elif plain:
            q = quantize_mx(x, "e4m3")
        out = ops.mx_linear_fast(q.data, q.scales, q.format, weight.data, weight.scales, k, residual, float(scale), out_dtype)
    return out if len(shape) == 2 else out.view(shape)
