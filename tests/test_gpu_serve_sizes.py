"""The 4-bit serving operators at the largest sizes that their documentation allows, against the same calls on parts of the input."""

from __future__ import annotations

import pytest
import torch

from mamba3_amd import MXTensor, _native, mx_linear, quantize_mx, sample_tokens

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _native_loaded(cuda_device):
    _native.lib()


@torch.no_grad()
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("each", [False, True])
def test_more_rows_than_a_grid_has_room_for(each, dtype):
    """A block of 1024 threads a row: from 2^22 rows on that is 2^32 threads."""
    rows, vocab, some = (1 << 22) + (1 << 21) + 5, 3, 1000
    gen = torch.Generator("cuda").manual_seed(0)
    z, u = torch.randn(rows, vocab, device="cuda", generator=gen).to(dtype), torch.rand(rows, device="cuda", generator=gen)
    settings = (0.7, 2, 0.9, 0.05)
    if each:
        r = [torch.rand(rows, device="cuda", generator=gen) for _ in range(4)]
        settings = (r[0] + 0.1, (r[1] * 4).int(), r[2], r[3] * 0.2)
    tokens, lp = sample_tokens(z, u, *settings, return_logprob=True)
    for at in (0, (1 << 21) - some // 2, (1 << 22) - some // 2, rows - some):
        part = slice(at, at + some)
        want = sample_tokens(z[part], u[part], *(v[part] if each else v for v in settings), return_logprob=True)
        assert torch.equal(tokens[part], want[0]) and torch.equal(lp[part], want[1])
    assert ((tokens >= 0) & (tokens < vocab)).all() and torch.isfinite(lp).all()


@torch.no_grad()
@pytest.mark.parametrize("rows,n", [(40, 1 << 25), (70, (1 << 25) + 70), (3, (1 << 26) - 5)])
def test_more_columns_than_tiles_take(rows, n):
    """From 2^25 columns on, 32 rows of bf16 results reach the end of what a descriptor bounds."""
    k, gen = 100, torch.Generator("cuda").manual_seed(0)
    w = MXTensor(torch.randint(256, (n, 64), device="cuda", generator=gen, dtype=torch.uint8),
                 torch.randint(120, 130, (n, 4), device="cuda", generator=gen, dtype=torch.uint8), (n, k), "e2m1")
    x = torch.randn(rows, k, device="cuda", generator=gen).bfloat16()
    res = torch.empty(rows, n, device="cuda", dtype=torch.bfloat16).normal_(generator=gen)
    for given in (x, quantize_mx(x, "e4m3")):
        y = mx_linear(given, w, res, 0.5)
        for at in (0, 1 << 24, n - 333):
            part = slice(at, at + 333)
            want = mx_linear(given, MXTensor(w.data[part], w.scales[part], (333, k), "e2m1"), res[:, part], 0.5)
            assert torch.equal(y[:, part], want)
