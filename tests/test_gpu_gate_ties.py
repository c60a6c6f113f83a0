"""The gate in front of microscaled values: elements lie on the side of a tie where the formula in 64 bits has them."""

from __future__ import annotations

import pytest
import torch

from mamba3_amd import _native, mx_linear, quantize_mx, silu_mul_mx

pytestmark = pytest.mark.gpu

LARGEST = {"e2m1": 6.0, "e4m3": 448.0}


@pytest.fixture(scope="module", autouse=True)
def _native_loaded(cuda_device):
    _native.lib()


def grid(fmt):
    if fmt == "e2m1":
        return torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device="cuda")
    return torch.arange(127, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn).double()


def silu(g):
    return g / (1 + torch.exp(-g))


def next_to_ties(fmt, rows, dtype, seed):
    """gate_up (rows, 64) of blocks with a scale of 1 whose other 31 products lie within a few steps of the inputs' type from ties,
    and the products in 64 bits."""
    gen = torch.Generator("cuda").manual_seed(seed)
    pts = grid(fmt)
    ties = (pts[1:] + pts[:-1]) / 2
    want = ties[torch.randint(len(ties), (rows, 32), device="cuda", generator=gen)] * (1 - 2 * torch.randint(2, (rows, 32), device="cuda", generator=gen))
    g = (torch.randn(rows, 32, device="cuda", generator=gen, dtype=torch.float64) * 4).to(dtype)
    g = torch.where(g.abs() < 2.0 ** -6, torch.ones_like(g), g)
    u = (want / silu(g.double())).to(dtype)
    g[:, 0], u[:, 0] = 32.0, LARGEST[fmt] / 32  # the largest element, so that the scale is 1
    return torch.cat([g, u], 1), silu(g.double()) * u.double()


@torch.no_grad()
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_products_next_to_ties(fmt, dtype):
    x, h = next_to_ties(fmt, 200_000, dtype, 0)
    pts = grid(fmt)
    at = torch.searchsorted((pts[1:] + pts[:-1]) / 2, h.abs())
    t = silu_mul_mx(x, fmt)
    assert (t.scales[:, 0] == 127).all()
    got = t.dequantize(torch.float32).double()
    off = (h.abs()[..., None] - ((pts[1:] + pts[:-1]) / 2)).abs().amin(-1) / h.abs()
    # the kernel's product is within 2^-34 of the exact one, the reference's within 2^-48
    sure = off > 2.0 ** -33
    assert sure.double().mean() > (0.99 if dtype == torch.float32 else 0.9)
    assert (off < 2.0 ** -21).sum() > (1_000_000 if dtype == torch.float32 else 10)  # where fp32 does not tell
    assert torch.equal(got[sure], torch.copysign(pts[at], h)[sure])


@torch.no_grad()
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_products_of_the_same_rows_in_one_launch(dtype):
    """The product that gates its rows itself sees the same elements."""
    x, _ = next_to_ties("e4m3", 96, dtype, 1)
    x = x.view(6, 16, 2, 32).transpose(1, 2).reshape(6, 1024)  # the blocks' gates, then their ups
    w = quantize_mx(torch.randn(40, 512, device="cuda", generator=torch.Generator("cuda").manual_seed(2)))
    assert torch.equal(mx_linear(x, w, gated=True), mx_linear(silu_mul_mx(x), w, out_dtype=dtype))


@torch.no_grad()
def test_gates_of_any_size():
    """Gates whose exponential vanishes or passes the largest number, infinities and NaN, rows of zeros."""
    g = torch.tensor([80.0, -80.0, 87.5, -87.5, -89.0, -95.0, -103.0, -104.5, 300.0, 3e38, 1e20, -1e20, 1e-30, -1e-30, 0.0, -0.0, 17.5, -17.5, 79.9, -79.9], device="cuda")
    u = torch.tensor([1.5, -1.0, 0.75, 3e37], device="cuda")
    gu = torch.cartesian_prod(g, u)
    x = torch.zeros(len(gu), 64, device="cuda")
    x[:, 3], x[:, 35] = gu[:, 0], gu[:, 1]  # a block each
    got = silu_mul_mx(x).dequantize(torch.float32).double()
    h = gu[:, 0].double() * torch.exp(torch.nn.functional.logsigmoid(gu[:, 0].double())) * gu[:, 1].double()
    past = h.abs() > torch.finfo(torch.float32).max
    assert past.any() and torch.isnan(got[past]).all() and torch.isfinite(got[~past]).all()
    # half a step of an element, and of the smallest one under the smallest scale
    assert ((got[:, 3] - h).abs()[~past] <= 2.0 ** -4 * h.abs()[~past] + 2.0 ** -137).all()
    assert (got[~past][:, [0, 1, 2, 4, 31]] == 0).all()
    bad = torch.zeros(4, 64, device="cuda")
    bad[0, 3], bad[1, 3], bad[2, 3], bad[:, 35] = float("inf"), float("nan"), -float("inf"), 1.0
    assert torch.isnan(silu_mul_mx(bad).dequantize()[:3]).all() and (silu_mul_mx(bad).dequantize()[3] == 0).all()


@torch.no_grad()
@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_far_negative_gates_beside_others(fmt):
    """Gates below -80 next to products of any size, up to factors that bring them back."""
    gen = torch.Generator("cuda").manual_seed(3)
    rows = 20_000
    g = torch.randn(rows, 32, device="cuda", generator=gen, dtype=torch.float64) * 60
    u = torch.randn(rows, 32, device="cuda", generator=gen, dtype=torch.float64) * torch.exp2(torch.randint(-60, 100, (rows, 1), device="cuda", generator=gen).double())
    far = torch.rand(rows, 1, device="cuda", generator=gen) < 0.3
    g = torch.where(far, -80 - 20 * torch.rand(rows, 32, device="cuda", generator=gen, dtype=torch.float64), g).float()  # rows that hold nothing else
    u = u.float()
    h = g.double() * torch.exp(torch.nn.functional.logsigmoid(g.double())) * u.double()
    t = silu_mul_mx(torch.cat([g, u], 1), fmt)
    got, scale = t.dequantize(torch.float32).double(), torch.exp2(t.scales[:, :1].double() - 127)
    # half a step: of an element 2^-4 (e4m3) or 2^-2 of it, of the smallest ones 2^-10 or 2^-2 of the scale
    off = 2.0 ** -4 * h.abs() + 2.0 ** -10 * scale if fmt == "e4m3" else 2.0 ** -2 * h.abs() + 2.0 ** -2 * scale
    assert ((got - h).abs() <= off * (1 + 2.0 ** -20) + 2.0 ** -148).all()
    top = h.abs().amax(1)
    last = 464.0 if fmt == "e4m3" else 7.0
    # the smallest scale under which the largest product rounds to an element
    sure = (top > 2.0 ** -110)
    assert (top <= last * scale[:, 0] * (1 + 2.0 ** -20))[sure].all() and (top >= last / 2 * scale[:, 0] * (1 - 2.0 ** -20))[sure].all()
