"""Operators that serve a model from 4-bit weights, against plain implementations in 64 bits: microscaled
quantisation and products, the residual's addition with its norm, the choice of the next token."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import mamba3_amd
from mamba3_amd import MXTensor

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16]
GRID = {"e2m1": torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64),
        "e4m3": torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()}
PAST = {"e2m1": 7.0, "e4m3": 464.0}  # what lies above rounds past the largest element (7 itself does: ties to even)


def half(t):
    """The largest relative error of one rounding."""
    return torch.finfo(t).eps / 2


def ref_blocks(x, fmt):
    """x (rows, k) in 64 bits -> (elements (rows, kp), exponents (rows, kp / 32), None where a block is not finite)."""
    rows, k = x.shape
    kp = -(-k // 128) * 128
    b = torch.zeros(rows, kp, dtype=torch.float64)
    b[:, :k] = x
    b = b.view(rows, kp // 32, 32)
    fine = torch.isfinite(b).all(-1)
    b = torch.where(fine[..., None], b, 0.0)
    top = b.abs().amax(-1)
    e = torch.zeros_like(top)
    some = top > 0
    low = torch.full_like(top, -127.0)
    # the smallest exponent from -127 on under which the largest magnitude is not past the grid
    for _ in range(260):
        v = top / torch.exp2(low)
        past = (v >= 7.0) if fmt == "e2m1" else (v > 464.0)
        low = torch.where(past, low + 1, low)
    e = torch.where(some, low, e)
    v = b / torch.exp2(e)[..., None]
    g = GRID[fmt]
    at = torch.searchsorted((g[1:] + g[:-1]) / 2, v.abs())
    mid = torch.cat([(g[1:] + g[:-1]) / 2, torch.tensor([math.inf], dtype=torch.float64)])[at]
    q = torch.copysign(g[torch.where((v.abs() == mid) & (at % 2 == 1), at + 1, at)], v)
    return q.view(rows, kp), e, fine


def ref_values(x, fmt):
    q, e, fine = ref_blocks(x, fmt)
    v = q.view(*e.shape, 32) * torch.exp2(e)[..., None]
    return torch.where(fine[..., None], v, math.nan).view(q.shape)[:, :x.shape[1]]


def stored_elements(t: MXTensor):
    data = t.data.cpu()
    if t.format == "e4m3":
        return data.view(torch.float8_e4m3fn).double()
    code = torch.stack((data & 15, data >> 4), -1).flatten(-2).long()
    return GRID["e2m1"][code & 7] * (1 - 2 * (code >> 3))


def gen(seed):
    return torch.Generator().manual_seed(seed)


def normal(shape, seed, dtype=torch.float32, std=1.0):
    return (torch.randn(shape, generator=gen(seed), dtype=torch.float64) * std).to(dtype)


# ------------------------------------------------------------------ quantisation
@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 7), (2, 31), (5, 32), (4, 33), (7, 127), (3, 128), (2, 129), (9, 500), (33, 1024), (2, 4099)])
def test_quantize(rows, k, dtype, fmt):
    x = normal((rows, k), rows * 1000 + k, dtype) * torch.exp(normal((rows, 1), k)).to(dtype)
    t = mamba3_amd.quantize_mx(x.cuda(), fmt)
    q, e, fine = ref_blocks(x.double(), fmt)
    assert t.shape == x.shape and t.format == fmt
    assert torch.equal(stored_elements(t), q)                      # zeros behind k too
    assert torch.equal(t.scales.cpu().double(), e + 127)
    v = ref_values(x.double(), fmt)
    assert torch.equal(t.dequantize(torch.float32).cpu().double(), v)
    assert torch.equal(t.dequantize().cpu().double(), v)           # four significant bits: exact in bf16


@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
def test_quantize_borders(fmt):
    """Every midpoint of the grid and what lies next to it, largest magnitudes around where the exponent steps, zeros,
    the smallest and the largest numbers."""
    rows = []
    last = GRID[fmt][-1].item()
    g = GRID[fmt]
    mids = ((g[1:] + g[:-1]) / 2).tolist()
    near = [f(m) for m in mids for f in (lambda v: v, lambda v: float(np.nextafter(np.float32(v), np.float32(0))),
                                         lambda v: float(np.nextafter(np.float32(v), np.float32(1e9))))]
    for i in range(0, len(near), 31):
        rows.append([last] + [(-1) ** j * v for j, v in enumerate(near[i:i + 31])])
    p = PAST[fmt]
    for s in (1.0, 2.0 ** -20, 2.0 ** 60):
        for top in (last, p, float(np.nextafter(np.float32(p), np.float32(0))), float(np.nextafter(np.float32(p), np.float32(1e9))), 2 * last):
            rows.append([top * s, last * s / 3, -p * s / 2, 0.1 * s])
    rows += [[0.0] * 32, [-0.0] * 5, [1e-45, -1e-45], [1.1754944e-38], [2.0 ** -127, 2.0 ** -126, 3e-39], [3.0e38, 1.0], [2.0 ** 120]]
    x = torch.zeros(len(rows), 32)
    for i, r in enumerate(rows):
        x[i, :len(r)] = torch.tensor(r, dtype=torch.float64).float()
    t = mamba3_amd.quantize_mx(x.cuda(), fmt)
    q, e, _ = ref_blocks(x.double(), fmt)
    assert torch.equal(t.scales.cpu().double(), e + 127)
    assert torch.equal(stored_elements(t), q)
    assert torch.equal(t.dequantize(torch.float32).cpu().double(), ref_values(x.double(), fmt).float().double())


@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_infinities_and_nan(dtype, fmt):
    x = normal((4, 96), 5, dtype)
    x[0, 40], x[1, 3], x[1, 70], x[2, 95] = math.inf, math.nan, -math.inf, -math.inf
    t = mamba3_amd.quantize_mx(x.cuda(), fmt)
    v = t.dequantize().cpu().double()
    want = ref_values(x.double(), fmt)
    assert torch.equal(torch.isnan(v), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(v), torch.nan_to_num(want))
    assert torch.isnan(want).any(0).sum() == 96 and (~torch.isnan(want[3])).all()


@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 50), (8, 128), (5, 333), (17, 2112)])
def test_silu_mul(rows, k, dtype, fmt):
    x = normal((rows, 2 * k), k, dtype, 2.0)
    x[0, 0], x[0, k] = -100.0, 3.0  # a gate whose exponential overflows: -0 or a number near it
    t = mamba3_amd.silu_mul_mx(x.cuda(), fmt)
    assert t.shape == (rows, k)
    g, u = x.double().chunk(2, 1)
    h = g / (1 + torch.exp(-g)) * u
    # fp32: exp, the sum, the quotient and the product are off by a few 2^-24 each
    off = 2.0 ** -20
    low, high = ref_values(h * (1 - off), fmt), ref_values(h * (1 + off), fmt)
    v = t.dequantize(torch.float32).cpu().double()
    near = ref_values(h, fmt)
    same = (low == high)
    assert same.double().mean() > 0.99
    assert torch.equal(v[same], near[same])
    assert ((v == low) | (v == high) | (v == near)).all()


def test_quantize_views_and_empty():
    x = normal((6, 4, 70), 3).cuda()
    want = mamba3_amd.quantize_mx(x.contiguous(), "e4m3").dequantize()
    for y in (x.transpose(0, 1).contiguous().transpose(0, 1), torch.cat([x, x], -1)[..., :70]):
        assert not y.is_contiguous()
        assert torch.equal(mamba3_amd.quantize_mx(y, "e4m3").dequantize(), want)
    odd = torch.empty(6 * 4 * 70 + 1, device="cuda")[1:].view(6, 4, 70).copy_(x)  # 4-byte aligned only
    assert torch.equal(mamba3_amd.quantize_mx(odd, "e4m3").dequantize(), want)
    none = mamba3_amd.quantize_mx(x[:0], "e2m1")
    assert none.shape == (0, 4, 70) and none.dequantize().shape == (0, 4, 70)


# ------------------------------------------------------------------ the residual's addition with the norm
def norm_sizes():
    return [(1, 1), (2, 5), (3, 8), (1, 64), (5, 129), (7, 500), (33, 512), (6, 513), (4, 1000), (9, 1024), (3, 1030), (5, 2048),
            (3, 2049), (2, 4096), (3, 5001), (2, 8192), (2, 8193), (1, 20000)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,d", norm_sizes())
def test_add_rms_norm(rows, d, dtype):
    x, r, w = normal((rows, d), 1, dtype), normal((rows, d), 2, dtype, 3.0), normal((d,), 3, dtype)
    dt, dy = normal((rows, d), 4, dtype), normal((rows, d), 5, dtype)
    scale, eps = 0.3, 1e-5
    ins = [t.cuda().requires_grad_() for t in (x, r, w)]
    total, y = mamba3_amd.add_rms_norm(*ins, scale, eps)
    grads = torch.autograd.grad([total, y], ins, [dt.cuda(), dy.cuda()])
    with torch.no_grad():
        again = mamba3_amd.add_rms_norm(*ins, scale, eps)
    assert torch.equal(again[0], total) and torch.equal(again[1], y)
    sum64 = r.double() + scale * x.double()
    assert ((total.cpu().double() - sum64).abs() <= half(dtype) * sum64.abs() + 2.0 ** -22 * (r.abs() + x.abs()).double()).all()
    t, w64, dy64, dt64 = total.detach().cpu().double(), w.double(), dy.double(), dt.double()
    rs = 1 / torch.sqrt(t.square().mean(1, keepdim=True) + eps)
    want = t * rs * w64
    small = 2.0 ** -20  # fp32 sums and products
    assert ((y.detach().cpu().double() - want).abs() <= (half(dtype) + small) * want.abs()).all()
    g = dy64 * w64
    dot = (g * t).sum(1, keepdim=True)
    d64 = dt64 + rs * g - t * rs ** 3 * dot / d
    size = dt64.abs() + rs * g.abs() + t.abs() * rs ** 3 * (g * t).abs().sum(1, keepdim=True) / d
    for got, s in ((grads[1], 1.0), (grads[0], scale)):
        assert ((got.cpu().double() - s * d64).abs() <= half(dtype) * (s * d64).abs() + small * s * size).all()
    parts = dy64 * t * rs
    dw = parts.sum(0)
    assert ((grads[2].cpu().double() - dw).abs() <= half(dtype) * dw.abs() + (small + rows * 2.0 ** -24) * parts.abs().sum(0)).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,d", [(9001, 41), (9002, 42), (9003, 43), (9004, 44), (9005, 45), (9006, 46), (9007, 47), (8300, 513),
                                    (4999, 767), (4100, 1027), (1700, 2051), (1601, 4094), (1100, 4099), (1050, 8190)])
def test_add_rms_norm_of_more_rows_than_run_at_once(rows, d, dtype):
    x, r, w = normal((rows, d), 1, dtype).cuda(), normal((rows, d), 2, dtype, 3.0).cuda(), normal((d,), 3, dtype).cuda()
    dt, dy = normal((rows, d), 4, dtype).cuda(), normal((rows, d), 5, dtype).cuda()
    ins = [t.requires_grad_() for t in (x, r, w)]
    total, y = mamba3_amd.add_rms_norm(*ins, 0.3, 1e-5)
    dx, dr, dw = torch.autograd.grad([total, y], ins, [dt, dy])
    t, w64, dy64, dt64 = total.detach().double(), w.detach().double(), dy.double(), dt.double()
    rs = 1 / torch.sqrt(t.square().mean(1, keepdim=True) + 1e-5)
    sum64 = r.detach().double() + 0.3 * x.detach().double()
    assert ((t - sum64).abs() <= half(dtype) * sum64.abs() + 2.0 ** -22 * (r.detach().abs() + x.detach().abs()).double()).all()
    y64 = t * rs * w64
    assert ((y.detach().double() - y64).abs() <= (half(dtype) + 2.0 ** -20) * y64.abs()).all()
    g = dy64 * w64
    d64 = dt64 + rs * g - t * rs ** 3 * (g * t).sum(1, keepdim=True) / d
    size = dt64.abs() + rs * g.abs() + t.abs() * rs ** 3 * (g * t).abs().sum(1, keepdim=True) / d
    small = 2.0 ** -20  # fp32 sums and products
    for got, s in ((dr, 1.0), (dx, 0.3)):
        assert ((got.double() - s * d64).abs() <= half(dtype) * (s * d64).abs() + small * s * size).all()
    parts = dy64 * t * rs
    want = parts.sum(0)
    assert ((dw.double() - want).abs() <= half(dtype) * want.abs() + (small + rows * 2.0 ** -24) * parts.abs().sum(0)).all()


@pytest.mark.parametrize("which", ["total", "y", "x", "residual", "weight"])
def test_add_rms_norm_one_result_or_one_gradient(which):
    x, r, w = (normal(s, i, torch.float32).cuda() for i, s in enumerate([(3, 70), (3, 70), (70,)]))
    ins = {"x": x, "residual": r, "weight": w}
    if which in ins:
        ins[which].requires_grad_()
        total, y = mamba3_amd.add_rms_norm(x, r, w, 0.5)
        (total * 2 + y * 3).sum().backward()
    else:
        for t in ins.values():
            t.requires_grad_()
        total, y = mamba3_amd.add_rms_norm(x, r, w, 0.5)
        (total if which == "total" else y).square().sum().backward()
    c = {k: v.detach().double().requires_grad_(v.requires_grad) for k, v in ins.items()}
    t64 = c["residual"] + 0.5 * c["x"]
    y64 = t64 * torch.rsqrt(t64.square().mean(1, keepdim=True) + 1e-5) * c["weight"]
    loss = (t64 * 2 + y64 * 3).sum() if which in ins else (t64 if which == "total" else y64).square().sum()
    loss.backward()
    for k, v in ins.items():
        if v.requires_grad:
            want = c[k].grad if c[k].grad is not None else torch.zeros_like(c[k])
            # 70 terms of size below 30 in fp32
            assert (v.grad.double() - want).abs().max() <= 70 * 30 * 2.0 ** -22


def test_add_rms_norm_against_differences():
    x, r, w = (normal(s, 40 + i, torch.float32).cuda() for i, s in enumerate([(4, 200), (4, 200), (200,)]))
    a, b = normal((4, 200), 50).cuda().double(), normal((4, 200), 51).cuda().double()

    def loss(x, r, w):
        total, y = mamba3_amd.add_rms_norm(x, r, w, 0.7)
        return (total.double() * a).sum() + (y.double() * b).sum()

    ins = [t.clone().requires_grad_() for t in (x, r, w)]
    loss(*ins).backward()
    h = 2.0 ** -6
    for i, t in enumerate(ins):
        v = normal(t.shape, 60 + i).cuda()
        up, down = ([q + s * h * v if j == i else q for j, q in enumerate((x, r, w))] for s in (1, -1))
        with torch.no_grad():
            slope = (loss(*up) - loss(*down)) / (2 * h)
        want = (t.grad.double() * v.double()).sum()
        # 1600 results rounded to 2^-24 of a few units, over 2 h; third derivatives times h^2 / 6
        assert abs(slope - want) <= 1600 ** 0.5 * 8 * 2.0 ** -24 / (2 * h) * 4 + 40 * h * h


@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("rows,d", norm_sizes())
def test_add_rms_norm_mx(rows, d, residual, dtype, fmt):
    x, r, w = normal((rows, d), 1, dtype), normal((rows, d), 2, dtype, 3.0), normal((d,), 3, dtype)
    total, q = mamba3_amd.add_rms_norm_mx(x.cuda(), r.cuda() if residual else None, w.cuda(), 0.3, 1e-5, fmt)
    if residual:
        assert torch.equal(total, mamba3_amd.add_rms_norm(x.cuda(), r.cuda(), w.cuda(), 0.3, 1e-5)[0])
    t = total.cpu().double()
    y = t / torch.sqrt(t.square().mean(1, keepdim=True) + 1e-5) * w.double()
    off = 2.0 ** -20
    low, high, near = (ref_values(y * f, fmt) for f in (1 - off, 1 + off, 1))
    v = q.dequantize(torch.float32).cpu().double()
    assert ((v == low) | (v == high) | (v == near)).all()
    assert q.scales.shape == (rows, -(-d // 128) * 4)
    assert (stored_elements(q)[:, d:] == 0).all()


def test_add_rms_norm_rows_of_zeros_and_infinities():
    x = torch.zeros(4, 96)
    x[1, 5], x[2, 5] = math.inf, math.nan
    x[3] = 1e-30
    w = torch.ones(96)
    total, y = mamba3_amd.add_rms_norm(x.cuda(), torch.zeros(4, 96).cuda(), w.cuda(), 1.0, 0.0)
    y = y.cpu()
    assert torch.isnan(y[0]).all()          # 0 / 0 without an eps
    assert torch.isnan(y[1, 5]) and (y[1, :5] == 0).all()
    assert torch.isnan(y[2]).all()
    total, q = mamba3_amd.add_rms_norm_mx(x.cuda(), None, w.cuda(), 1.0, 1e-5)
    v = q.dequantize().cpu()
    assert (v[0] == 0).all()
    assert torch.isnan(v[1, :32]).all() and (v[1, 32:] == 0).all() and torch.isnan(v[2]).all()


# ------------------------------------------------------------------ products
def mx_pair(rows, n, k, fmt, seed):
    x = normal((rows, k), seed) * torch.exp(normal((rows, 1), seed + 1))
    w = normal((n, k), seed + 2, std=0.05)
    return mamba3_amd.quantize_mx(x.cuda(), fmt), mamba3_amd.quantize_mx(w.cuda(), "e2m1")


def product_bounds(x: MXTensor, w: MXTensor):
    """The product in 64 bits; how far its sums may be off for a bf16 result (e4m3: 2^-11 of the largest product in each
    128 that are added at once) and for an fp32 one (a rounding of the running sum for each product)."""
    a, b = x.dequantize(torch.float32).cpu().double(), w.dequantize(torch.float32).cpu().double()
    p = (a.abs()[:, None, :] * b.abs()[None])
    size = p.sum(-1)
    k = p.shape[-1]
    pad = torch.nn.functional.pad(p, (0, -k % 128)).unflatten(-1, (-1, 128)).amax(-1).sum(-1)
    step = 2.0 ** -11 * pad if x.format == "e4m3" else 0.0
    return a @ b.t(), step + k * 2.0 ** -24 * size, k * 2.0 ** -24 * size


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (1, 16, 128), (2, 5, 33), (4, 100, 300), (8, 48, 512), (15, 17, 129), (16, 64, 256), (17, 33, 640),
                                      (31, 65, 96), (33, 40, 500), (64, 130, 384), (65, 70, 200), (100, 129, 257), (130, 257, 129)])
def test_mx_linear(rows, n, k, dtype, fmt):
    x, w = mx_pair(rows, n, k, fmt, rows + n + k)
    want, off16, off32 = product_bounds(x, w)
    y = mamba3_amd.mx_linear(x, w, out_dtype=dtype)
    assert y.shape == (rows, n) and y.dtype == dtype
    off = off16 if dtype == torch.bfloat16 else off32
    assert ((y.cpu().double() - want).abs() <= half(dtype) * want.abs() + off).all()
    r = normal((rows, n), 9, dtype)
    y = mamba3_amd.mx_linear(x, w, r.cuda(), 0.25).cpu().double()
    want = r.double() + 0.25 * want
    assert ((y - want).abs() <= half(dtype) * want.abs() + 0.25 * off + 2.0 ** -23 * want.abs()).all()


@pytest.mark.parametrize("rows,n,k", [(300, 300, 1024), (513, 257, 2176), (1000, 770, 500), (257, 1030, 768)])
@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_mx_linear_many_rows(rows, n, k, dtype, fmt):
    x, w = mx_pair(rows, n, k, fmt, 7)
    a, b = x.dequantize(torch.float32).double(), w.dequantize(torch.float32).double()
    want, size = a @ b.t(), a.abs() @ b.abs().t()
    # the largest product of 128 is at most the largest factors'
    top = lambda v: torch.nn.functional.pad(v.abs(), (0, -k % 128)).unflatten(-1, (-1, 128)).amax(-1)  # noqa: E731
    step = 2.0 ** -11 * (top(a) @ top(b).t()) if fmt == "e4m3" and dtype == torch.bfloat16 else 0.0
    y = mamba3_amd.mx_linear(x, w, out_dtype=dtype)
    assert ((y.double() - want).abs() <= half(dtype) * want.abs() + step + k * 2.0 ** -24 * size).all()
    r = normal((rows, n), 3, dtype).cuda()
    assert ((mamba3_amd.mx_linear(x, w, r, -2.0).double() - (r.double() - 2 * want)).abs()
            <= half(dtype) * (r.double() - 2 * want).abs() + 2 * step + 2.0 ** -22 * (r.abs().double() + 2 * want.abs()) + 2 * k * 2.0 ** -24 * size).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 3, 8, 16, 20, 70, 300])
def test_mx_linear_of_a_tensor_is_that_of_its_quantisation(rows, dtype):
    w = mamba3_amd.quantize_mx(normal((90, 330), 1).cuda())
    x = normal((rows, 330), 2, dtype).cuda()
    y = mamba3_amd.mx_linear(x, w)
    assert y.dtype == dtype
    assert torch.equal(y, mamba3_amd.mx_linear(mamba3_amd.quantize_mx(x, "e4m3"), w, out_dtype=dtype))
    three = mamba3_amd.mx_linear(x.view(rows, 1, 330), w)
    assert three.shape == (rows, 1, 90) and torch.equal(three.view(rows, 90), y)


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 20, 150])
def test_mx_linear_not_a_number_stays_in_its_row(rows, dtype, fmt):
    x = normal((rows, 200), 1)
    x[0, 150] = math.inf
    w = normal((50, 200), 2)
    w[7, 3] = math.nan
    y = mamba3_amd.mx_linear(mamba3_amd.quantize_mx(x.cuda(), fmt), mamba3_amd.quantize_mx(w.cuda()), out_dtype=dtype).cpu()
    assert torch.isnan(y[0]).all() and torch.isnan(y[:, 7]).all()
    y[0], y[:, 7] = 0, 0
    assert torch.isfinite(y).all()


def test_mx_linear_scales_far_apart():
    """Blocks whose powers of two lie at the ends of the range, with products of ordinary size."""
    x, w = torch.ones(3, 128), torch.ones(20, 128)
    for i, e in enumerate((100, -100, 60, -126)):
        x[:, 32 * i:32 * i + 32] *= 2.0 ** e
        w[:, 32 * i:32 * i + 32] *= 2.0 ** (-e if e != -126 else 120)
    for dtype in DTYPES:
        y = mamba3_amd.mx_linear(mamba3_amd.quantize_mx(x.cuda(), "e4m3"), mamba3_amd.quantize_mx(w.cuda()), out_dtype=dtype)
        assert torch.equal(y.cpu().double(), torch.full((3, 20), 32 * (3 + 2.0 ** -6), dtype=torch.float64).to(dtype).double())


def test_mx_linear_strided_residual_and_no_rows():
    x, w = mx_pair(6, 40, 96, "e4m3", 3)
    r = normal((6, 80), 4, torch.bfloat16).cuda()
    assert torch.equal(mamba3_amd.mx_linear(x, w, r[:, ::2]), mamba3_amd.mx_linear(x, w, r[:, ::2].contiguous()))
    assert mamba3_amd.mx_linear(torch.empty(0, 96, device="cuda", dtype=torch.bfloat16), w).shape == (0, 40)


def test_mx_linear_many_columns_and_a_long_row():
    """Weights past 2^31 bytes of offset would need 4 GB; this has rows past 2^16 columns and k of 2^14."""
    x, w = mx_pair(3, 70001, 128, "e4m3", 1)
    a, b = x.dequantize(torch.float32).double(), w.dequantize(torch.float32).double()
    y = mamba3_amd.mx_linear(x, w).double()
    assert ((y - a @ b.t()).abs() <= half(torch.bfloat16) * (a @ b.t()).abs() + (2.0 ** -11 + 128 * 2.0 ** -24) * (a.abs() @ b.abs().t())).all()
    x, w = mx_pair(5, 20, 1 << 14, "e4m3", 2)
    a, b = x.dequantize(torch.float32).double(), w.dequantize(torch.float32).double()
    y = mamba3_amd.mx_linear(x, w, out_dtype=torch.float32).double()
    assert ((y - a @ b.t()).abs() <= 2.0 ** -12 * 2.0 ** -10 * (a.abs() @ b.abs().t())).all()


# ------------------------------------------------------------------ the next token
def ref_sample(z, u, t=1.0, k=0, p=1.0, m=0.0):
    """(token, log probability, how near a border lies) of one row, from sorted masses in 64 bits."""
    z = np.where(np.isnan(z), -np.inf, z.astype(np.float64))
    v = len(z)
    order = np.lexsort((np.arange(v), -z))
    if z[order[0]] == -np.inf:
        return -1, math.nan, 1.0
    if not t > 0:
        return int(order[0]), 0.0, 1.0
    zs = z[order]
    with np.errstate(invalid="ignore"):
        gap = np.where(zs == zs[0], 0.0, zs - zs[0])
    mass = np.exp(gap / t)
    real = int((zs > -np.inf).sum())
    n = min(k, real) if k > 0 else real
    near = 1.0
    cum = np.cumsum(mass[:n])
    if p < 1:
        goal = p * cum[-1]
        last = int(np.searchsorted(cum, goal)) if p > 0 else 0
        near = min(near, np.abs(cum - goal).min() / cum[-1]) if p > 0 else near
        n = min(n, last + 1)
    n = max(1, min(n, int((mass >= min(m, 1.0)).sum())))
    if m > 0:
        near = min(near, np.abs(mass[mass < 1] - m).min(initial=1.0))  # a mass of 1 is exact
    cum = cum[:n]
    goal = min(max(u, 0.0), 1 - 2.0 ** -30) * cum[-1]
    at = min(int(np.searchsorted(cum, goal, side="right")), n - 1)
    if u > 0:  # the last kept token's end is no border: u is below 1, or taken there
        near = min(near, np.abs(cum[:-1] - goal).min(initial=cum[-1]) / cum[-1])
    return int(order[at]), gap[at] / t - math.log(cum[-1]), near


def check_sample(z, u, **kw):
    """Tokens and log probabilities of all rows; rows nearer to a border than 1e-8 of the mass may fall either way."""
    rows = z.shape[0]
    to = lambda v: v.cuda() if torch.is_tensor(v) else v  # noqa: E731
    token, lp = mamba3_amd.sample_tokens(z.cuda(), u.cuda(), *[to(kw.get(n, d)) for n, d in (("t", 1.0), ("k", 0), ("p", 1.0), ("m", 0.0))], return_logprob=True)
    alone = mamba3_amd.sample_tokens(z.cuda(), u.cuda(), *[to(kw.get(n, d)) for n, d in (("t", 1.0), ("k", 0), ("p", 1.0), ("m", 0.0))])
    assert torch.equal(token, alone) and token.dtype == torch.int64
    checked = 0
    for i in range(rows):
        one = {n: (v[i].item() if torch.is_tensor(v) else v) for n, v in kw.items()}
        want, want_lp, near = ref_sample(z[i].float().numpy(), u[i].item(), **one)
        if near < 1e-8:
            continue
        checked += 1
        assert token[i].item() == want, (i, one, u[i].item())
        if math.isnan(want_lp):
            assert math.isnan(lp[i].item())
        else:
            assert abs(lp[i].item() - want_lp) <= 2.0 ** -22 * max(1.0, abs(want_lp))
    assert checked >= rows - max(1, rows // 3)  # equal logits put borders on exact shares


SETTINGS = [dict(), dict(t=0.0), dict(t=0.7, k=1), dict(k=5), dict(t=1.3, k=50, p=0.9), dict(p=0.5), dict(p=0.999), dict(p=0.0), dict(m=0.1), dict(m=1.0),
            dict(t=0.5, k=40, p=0.8, m=0.05), dict(t=3.0, p=0.95), dict(t=0.05, k=7), dict(k=10 ** 9, p=0.7, m=0.001)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1, 2, 7, 64, 500, 2047, 5003, 32000])
@pytest.mark.parametrize("setting", range(len(SETTINGS)))
def test_sample(setting, vocab, dtype):
    rows = 12 if vocab < 10000 else 4
    z = normal((rows, vocab), vocab, dtype, 2.5)
    z[0, vocab // 2] = 9.0
    if vocab > 4:
        z[1, 1::2] = -math.inf
        z[2, ::3] = math.nan
        z[3] = z[3, 0]  # all alike
    u = torch.rand(rows, generator=gen(setting))
    check_sample(z, u, **SETTINGS[setting])


def test_sample_settings_by_row():
    rows, vocab = 64, 3001
    z = normal((rows, vocab), 1, torch.float32, 3.0)
    r = lambda s: torch.rand(rows, generator=gen(s))  # noqa: E731
    t = torch.where(r(1) < 0.2, 0.0, 0.2 + r(2))
    k = torch.where(r(3) < 0.3, 0, (r(4) * 200).int() + 1)
    check_sample(z, r(5), t=t, k=k, p=0.3 + 0.75 * r(6), m=torch.where(r(7) < 0.5, 0.0, 0.2 * r(8)))
    check_sample(z, r(9), t=0.9, k=k.long(), p=0.9)


@pytest.mark.parametrize("dtype", DTYPES)
def test_sample_ends_of_u(dtype):
    z = normal((8, 1000), 2, dtype, 2.0)
    for v in (0.0, 1 - 2.0 ** -24, 1.0, 2.0, -1.0):
        check_sample(z, torch.full((8,), v), k=20, p=0.9)
    first = mamba3_amd.sample_tokens(z.cuda(), torch.full((8,), math.nan).cuda())
    assert torch.equal(first.cpu(), mamba3_amd.sample_tokens(z.cuda(), torch.zeros(8).cuda(), 0.0).cpu())


@pytest.mark.parametrize("kw", [dict(), dict(k=9000), dict(p=0.4), dict(k=12000, p=0.7), dict(m=0.5)])
def test_sample_many_equal_logits(kw):
    """More ties than are sorted at once, in one bin and over few values."""
    z = torch.zeros(6, 20000)
    z[1] = (torch.arange(20000) % 3).float()
    z[2] = (torch.arange(20000) % 5).float() / 256
    z[3] = -1000.0
    z[3, 17] = 0.0
    z[4] = normal((20000,), 4) * 2.0 ** -9        # one bin, all different
    z[5] = -500 + normal((20000,), 5)             # far behind one token: the last bin
    z[5, 3] = 3.0
    check_sample(z, torch.tensor([0.37, 0.5, 0.999, 0.1, 0.77, 0.9]), **kw)
    check_sample(z.bfloat16(), torch.tensor([0.37, 0.5, 0.999, 0.1, 0.77, 0.9]), **kw)


def test_sample_far_tail_counts():
    """top_k that ends far below the likeliest token, and temperatures that make the tail count."""
    z = normal((4, 6000), 6, torch.float32, 30.0)
    for kw in (dict(k=5000, t=100.0), dict(k=3000, t=50.0, p=0.99), dict(t=1000.0, p=0.5), dict(t=200.0, m=0.7)):
        check_sample(z, torch.tensor([0.9, 0.99, 0.5, 0.2]), **kw)


def test_sample_rows_without_a_token_and_infinities():
    z = torch.full((5, 300), -math.inf)
    z[1] = math.nan
    z[2, 7], z[2, 200] = math.inf, math.inf
    z[3, 299] = -3e38
    z[4, 5], z[4, 6] = -0.0, 0.0  # equal: the lower index first
    token, lp = mamba3_amd.sample_tokens(z.cuda(), torch.tensor([0.5, 0.5, 0.6, 0.5, 0.3]).cuda(), return_logprob=True)
    assert token.tolist() == [-1, -1, 200, 299, 5]
    assert torch.isnan(lp[:2]).all() and abs(lp[2].item() + math.log(2)) < 1e-6 and lp[3].item() == 0.0
    token = mamba3_amd.sample_tokens(z.cuda(), torch.full((5,), 0.9).cuda(), 0.0)
    assert token.tolist() == [-1, -1, 7, 299, 5]
    assert mamba3_amd.sample_tokens(z[:0].cuda(), torch.empty(0, device="cuda")).shape == (0,)


def test_sample_follows_the_masses():
    """Over evenly spread u, each token comes as often as its share of the kept mass says."""
    z = normal((1, 50), 3, torch.float32, 1.5)
    n = 20000
    u = (torch.arange(n) + 0.5) / n
    token = mamba3_amd.sample_tokens(z.expand(n, 50).cuda(), u.cuda(), 0.8, 20, 0.9).cpu()
    share = torch.softmax(z[0].double() / 0.8, 0)
    order = torch.argsort(share, descending=True)[:20]
    cum = share[order].cumsum(0)
    kept = order[:int((cum < 0.9 * cum[-1]).sum()) + 1]
    want = share[kept] / share[kept].sum()
    count = torch.bincount(token, minlength=50).double() / n
    assert (count[kept] - want).abs().max() <= 2 / n and abs(count.sum() - count[kept].sum()) == 0


@pytest.mark.parametrize("rows,n,k", [(33, 9999, 64), (40, 9304, 300), (50, 9222, 2050), (64, 9217, 129), (12, 25700, 1600), (25, 25704, 1100), (5, 65600, 2048)])
@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_mx_linear_few_rows_many_columns(rows, n, k, fmt):
    x, w = mx_pair(rows, n, k, fmt, 11)
    a, b = x.dequantize(torch.float32).double(), w.dequantize(torch.float32).double()
    want, size = a @ b.t(), a.abs() @ b.abs().t()
    top = lambda v: torch.nn.functional.pad(v.abs(), (0, -k % 128)).unflatten(-1, (-1, 128)).amax(-1)  # noqa: E731
    step = 2.0 ** -11 * (top(a) @ top(b).t()) if fmt == "e4m3" else 0.0
    off = step + k * 2.0 ** -24 * size
    assert ((mamba3_amd.mx_linear(x, w).double() - want).abs() <= half(torch.bfloat16) * want.abs() + off).all()
    r = normal((rows, n), 3, torch.bfloat16).cuda()
    want = r.double() - 0.75 * want
    assert ((mamba3_amd.mx_linear(x, w, r, -0.75).double() - want).abs()
            <= half(torch.bfloat16) * want.abs() + 0.75 * off + 2.0 ** -22 * (r.abs().double() + 2 * want.abs())).all()


@pytest.mark.parametrize("rows,n,k", [(256, 20001, 2000), (700, 7501, 2000), (1100, 9101, 1003), (8200, 9602, 130)])
@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_mx_linear_many_rows_fp32(rows, n, k, fmt):
    from mamba3_amd import _native
    assert _native._mx_exact_bytes(rows, n, k) > 0  # sizes that go by way of bf16 copies
    x, w = mx_pair(rows, n, k, fmt, 13)
    a, b = x.dequantize(torch.float32).double(), w.dequantize(torch.float32).double()
    want, size = a @ b.t(), a.abs() @ b.abs().t()
    off = k * 2.0 ** -24 * size
    y = mamba3_amd.mx_linear(x, w, out_dtype=torch.float32)
    assert y.dtype == torch.float32 and ((y.double() - want).abs() <= half(torch.float32) * want.abs() + off).all()
    r = normal((rows * n + 1,), 3).cuda()[1:].view(rows, n)  # four bytes past an aligned address
    want = r.double() + 0.25 * want
    assert ((mamba3_amd.mx_linear(x, w, r, 0.25).double() - want).abs() <= 2.0 ** -23 * (want.abs() + r.abs()) + 0.25 * off).all()
    x.scales[3, 0] = 255
    y = mamba3_amd.mx_linear(x, w, out_dtype=torch.float32)
    assert torch.isnan(y[3]).all() and torch.isfinite(y[:3]).all() and torch.isfinite(y[4:]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_add_rms_norm_mx_large_and_small_values(dtype):
    """Rows whose products with the weight alone would overflow or vanish; and each element on the side of a tie where the formula in
    64 bits has it."""
    x = normal((6, 384), 0, torch.float64) * torch.tensor([1e18, 1e-18, 1.0, 1e15, 1e-10, 3.0])[:, None].double()
    w = normal((384,), 1, torch.float64) * torch.tensor([1e22, 1e-20, 1.0]).repeat(128).double()
    x, w = x.to(dtype), w.to(dtype)
    q = mamba3_amd.add_rms_norm_mx(x.cuda(), None, w.cuda(), eps=1e-30)[1]
    t = x.double()
    y = t / torch.sqrt(t.square().mean(1, keepdim=True) + 1e-30) * w.double()
    assert torch.equal(q.dequantize(torch.float32).cpu().double(), ref_values(y, "e4m3").float().double())
    big = normal((3000, 512), 2, dtype)
    w = normal((512,), 3, dtype)
    for fmt in ("e4m3", "e2m1"):
        v = mamba3_amd.add_rms_norm_mx(big.cuda(), None, w.cuda(), 1.0, 1e-5, fmt)[1].dequantize(torch.float32).cpu().double()
        t = big.double()
        want = ref_values(t / torch.sqrt(t.square().mean(1, keepdim=True) + 1e-5) * w.double(), fmt)
        # a row's reciprocal root is 2^-28 or so from exact: of 1.5 million elements one may be that near to a tie
        assert (v != want).sum() <= 2


def test_add_rms_norm_mx_past_the_largest_number():
    x, w = normal((4, 128), 5), torch.full((128,), 2.5e38)
    w[64:] = 1.0
    y = (x.double() / torch.sqrt(x.double().square().mean(1, keepdim=True))) * w.double()
    past = (y.abs() > torch.finfo(torch.float32).max).view(4, 4, 32).any(-1)
    assert past.any() and not past.all()
    v = mamba3_amd.add_rms_norm_mx(x.cuda(), None, w.cuda(), eps=0.0)[1]
    assert torch.equal(v.scales.cpu() == 255, past)  # an infinity makes its block NaN


@pytest.mark.parametrize("rows,n,k", [(2100, 9000, 1600), (2100, 9001, 1600), (4000, 4616, 1536), (300, 40008, 1700)])
@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_mx_linear_rounds_of_tiles(rows, n, k, fmt):
    """Sizes whose last columns may go to other tiles than the rest."""
    x, w = mx_pair(rows, n, k, fmt, 17)
    a, b = x.dequantize(torch.float32).double(), w.dequantize(torch.float32).double()
    want, size = a @ b.t(), a.abs() @ b.abs().t()
    top = lambda v: torch.nn.functional.pad(v.abs(), (0, -k % 128)).unflatten(-1, (-1, 128)).amax(-1)  # noqa: E731
    off = k * 2.0 ** -24 * size + (2.0 ** -11 * (top(a) @ top(b).t()) if fmt == "e4m3" else 0.0)
    assert ((mamba3_amd.mx_linear(x, w).double() - want).abs() <= half(torch.bfloat16) * want.abs() + off).all()
    r = normal((rows, n), 3, torch.bfloat16).cuda()
    want = r.double() - 0.75 * want
    assert ((mamba3_amd.mx_linear(x, w, r, -0.75).double() - want).abs()
            <= half(torch.bfloat16) * want.abs() + 0.75 * off + 2.0 ** -22 * (r.abs().double() + 2 * want.abs())).all()
