"""How many digits the choice of the next token keeps: its log probability, and the masses that it compares u with."""

from __future__ import annotations

import math
from decimal import Decimal, getcontext

import pytest
import torch

from mamba3_amd import _native, sample_tokens

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _native_loaded(cuda_device):
    _native.lib()


@torch.no_grad()
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kw", [dict(), dict(top_k=2), dict(top_p=1 - 2.0 ** -40, min_p=1e-13)])
@pytest.mark.parametrize("vocab", [2, 1000, 128000])
def test_log_probability_of_one_likely_token(vocab, kw, dtype):
    """What the others add to its mass of 1 is what there is to know, however small."""
    gaps = torch.tensor([4.0, 8.0, 12.0, 16.0, 18.0, 20.0, 22.0, 24.0])
    z = torch.full((len(gaps), vocab), -float("inf"))
    z[:, 0], z[:, -1] = 3.0, 3.0 - gaps
    token, lp = sample_tokens(z.to(dtype).cuda(), torch.zeros(len(gaps), device="cuda"), return_logprob=True, **kw)
    assert (token == 0).all()
    want = -torch.log1p(torch.exp(-gaps.double()))
    # rounded to fp32 once; the other's mass, and that of all up to it, are whole numbers of 2^-shift, 62 less the bits of vocab or 51
    shift = min(62 - (vocab - 1).bit_length(), 51)
    assert ((lp.cpu().double() - want).abs() <= 2.0 ** -24 * want.abs() + 2 * 2.0 ** -shift + 2.0 ** -36 * torch.exp(-gaps.double())).all()


@torch.no_grad()
def test_log_probabilities_are_the_64_bit_ones_rounded():
    z = torch.randn(64, 5000, generator=torch.Generator().manual_seed(0)) * 4
    u = torch.rand(64, generator=torch.Generator().manual_seed(1))
    for kw in (dict(), dict(temperature=0.3), dict(temperature=2.0, top_k=300)):
        token, lp = sample_tokens(z.cuda(), u.cuda(), return_logprob=True, **kw)
        masses = z.double() / kw.get("temperature", 1.0)
        if "top_k" in kw:
            masses = masses.masked_fill(z < z.topk(kw["top_k"]).values[:, -1:], -float("inf"))
        want = torch.log_softmax(masses, 1).gather(1, token.cpu()[:, None])[:, 0]
        # a mass is off by 2^-36 of itself at most and by 2^-50
        assert ((lp.cpu().double() - want).abs() <= 2.0 ** -24 * want.abs() + 2.0 ** -35).all()


@torch.no_grad()
@pytest.mark.parametrize("vocab", [2, 1500])
@pytest.mark.parametrize("off", [6e-13, -6e-13])
def test_masses_next_to_a_border(off, vocab):
    """Two tokens, of masses 1 and m: u is just before or past the end of the first, 1 / (1 + m), by less than the fifth term of
    exp's series where m lies at the end of a bin (7.8e-12 of m, a quarter of that here)."""
    getcontext().prec = 40
    z = torch.full((8, vocab), -float("inf"))
    gap = 2.0 ** -6 + 2.0 ** -20 * torch.arange(8)
    z[:, 0], z[:, 1] = 0.0, -gap
    u, temperature, want = [], [], []
    for g in gap.tolist():
        one = torch.tensor(1 / (1 + math.exp(-1 / 64.001))).item()
        u.append(one)
        # the temperature that puts the border at u (1 + off): exp(-g / t) = 1 / border - 1
        border = Decimal(one) * (1 + Decimal(off))
        temperature.append(float(-Decimal(g) / (1 / border - 1).ln()))
        real = 1 / (1 + (-Decimal(g) / Decimal(temperature[-1])).exp())
        assert abs(real / border - 1) < Decimal("2e-16")
        want.append(1 if Decimal(one) >= real else 0)
    assert want == [0 if off > 0 else 1] * 8
    # the series to 2e-14 of m and whole numbers of 2^-51: 1e-14 of the whole
    got = [sample_tokens(z[i:i + 1].cuda(), torch.tensor(u[i:i + 1]).cuda(), t).item() for i, t in enumerate(temperature)]
    assert got == want
