"""The language model's 4-bit copies of its weights on the GPU: captured graphs and other streams that read them while they are
made anew."""

from __future__ import annotations

import pytest
import torch

from mamba3_amd import KulaMambaLM, _native, add_rms_norm_mx, mx_linear, quantize_mx

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _native_loaded(cuda_device):
    _native.lib()


def small_lm(vocab=500, d=128):
    torch.manual_seed(0)
    return KulaMambaLM(vocab, d, n_layers=1, d_state=32, headdim=32, mimo_rank=2).cuda().bfloat16().eval()


def rows(n, d, seed):
    return torch.randn(n, d, generator=torch.Generator().manual_seed(seed)).bfloat16().cuda()


def logits(lm, x):
    """By the operators one by one, from the head's weight as it is."""
    return mx_linear(add_rms_norm_mx(x, None, lm.norm.weight, eps=lm.norm.eps)[1], quantize_mx(lm.lm_head.weight.detach()), out_dtype=x.dtype)


@torch.no_grad()
def test_a_captured_graph_follows_a_second_quantisation():
    lm, x = small_lm().quantize_mx(), rows(2, 128, 0)
    lm._mx_logits(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = lm._mx_logits(x)
    for i in range(3):
        lm.lm_head.weight.data.mul_(1.5).add_(0.01 * i)  # leaves no trace
        lm.quantize_mx()
        junk = [torch.full((1 << 14,), 255, dtype=torch.uint8, device="cuda") for _ in range(64)]  # what freed memory would go to
        want = logits(lm, x)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        del junk


@torch.no_grad()
@pytest.mark.parametrize("captured", [False, True])
def test_weights_are_replaced_while_another_stream_reads_the_copy(captured):
    """The other stream's products, still waiting behind long work, keep the weights that they were launched with."""
    lm, x = small_lm(20000, 256).quantize_mx(), rows(64, 256, 0)
    if captured:
        lm._mx_logits(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = lm._mx_logits(x)
    side, long = torch.cuda.Stream(), torch.zeros(8192, 8192, device="cuda", dtype=torch.bfloat16)
    for i in range(3):
        old = lm.lm_head.weight
        first = logits(lm, x)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for _ in range(20):
                long = long @ long
            if captured:
                graph.replay()
                kept = got.clone()
            else:
                kept = lm._mx_logits(x)
        lm.lm_head.weight = torch.nn.Parameter(old.flip(0) * (1.5 + i))
        now = lm._mx_logits(x)
        torch.cuda.synchronize()
        assert torch.equal(kept, first) and torch.equal(now, logits(lm, x)) and not torch.equal(now, first)
        if captured:
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, now)
