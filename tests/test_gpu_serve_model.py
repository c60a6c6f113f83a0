"""The 4-bit serving operators as they are used: in front of one another, by the language model, in captured graphs,
on other streams and under torch.compile, at sizes past 32-bit offsets. What each computes is tested by itself elsewhere; here
results are compared with those of the same operators called one by one, bit for bit."""

from __future__ import annotations

import copy

import pytest
import torch
import torch.nn.functional as F

import mamba3_amd
from mamba3_amd import KulaMambaLM, _native, add_rms_norm, add_rms_norm_mx, mx_linear, quantize_mx, sample_tokens, silu_mul_mx

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(scope="module", autouse=True)
def _native_loaded(cuda_device):
    _native.lib()


def normal(shape, seed, dtype=torch.float32, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).cuda()


def same(a, b):
    return a.shape == b.shape and a.dtype == b.dtype and torch.equal(a, b)


# ---------------------------------------------------------------- what stands in front of a product
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (1, 300, 768), (2, 33, 31), (3, 64, 512), (4, 3696, 768), (5, 70, 513), (7, 17, 129), (9, 40, 1999), (15, 48, 2048),
                                      (16, 16, 2048), (16, 5000, 700), (17, 64, 768), (3, 64, 2049), (2, 20, 9000), (200, 300, 500)])
def test_norm_in_front_of_a_product(rows, n, k, dtype):
    x, nw = normal((rows, k), rows, dtype, 3.0), normal((k,), k, dtype)
    w, res = quantize_mx(normal((n, k), 1)), normal((rows, n), 2, dtype)
    q = add_rms_norm_mx(x, None, nw, eps=1e-3)[1]
    assert same(mx_linear(x, w, norm_weight=nw, eps=1e-3), mx_linear(q, w, out_dtype=dtype))
    assert same(mx_linear(x, w, res, 0.25, norm_weight=nw, eps=1e-3), mx_linear(q, w, res, 0.25))
    other = torch.float32 if dtype == torch.bfloat16 else torch.bfloat16
    assert same(mx_linear(x, w, out_dtype=other, norm_weight=nw, eps=1e-3), mx_linear(q, w, out_dtype=other))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (1, 768, 2112), (2, 33, 31), (4, 768, 2112), (5, 70, 513), (7, 17, 129), (15, 48, 2048), (16, 16, 2048),
                                      (17, 64, 768), (2, 20, 20000), (200, 300, 500)])
def test_gate_in_front_of_a_product(rows, n, k, dtype):
    x, w, res = normal((rows, 2 * k), rows, dtype, 3.0), quantize_mx(normal((n, k), 1)), normal((rows, n), 2, dtype)
    q = silu_mul_mx(x)
    assert same(mx_linear(x, w, gated=True), mx_linear(q, w, out_dtype=dtype))
    assert same(mx_linear(x, w, res, 0.25, gated=True), mx_linear(q, w, res, 0.25))


def test_in_front_of_a_product_odd_memory():
    x, w = normal((6, 2 * 70), 0)[::2, 3:73], quantize_mx(normal((9, 70), 1))
    nw = normal((140,), 2)[::2]
    assert same(mx_linear(x, w, norm_weight=nw), mx_linear(x.contiguous(), w, norm_weight=nw.contiguous()))
    xb = normal((3 * 71 + 1,), 4, torch.bfloat16)[1:].view(3, 71)  # two bytes past an aligned address
    wb = quantize_mx(normal((9, 71), 1))
    assert same(mx_linear(xb, wb, norm_weight=nw.bfloat16().new_ones(71)), mx_linear(xb.clone(), wb, norm_weight=nw.bfloat16().new_ones(71)))
    bad = normal((2, 64), 3, torch.bfloat16)
    bad[1, 7] = float("nan")
    y = mx_linear(bad, quantize_mx(normal((5, 64), 1)), norm_weight=bad.new_ones(64))
    assert torch.isfinite(y[0]).all() and torch.isnan(y[1]).all()


# ---------------------------------------------------------------- the language model
def small_lm(dtype=torch.bfloat16, **kw):
    torch.manual_seed(0)
    return KulaMambaLM(500, 128, n_layers=2, d_state=32, headdim=32, mimo_rank=2, **kw).cuda().to(dtype).eval()


def by_hand(lm, ids):
    """Logits, from the operators one by one."""
    x = lm.embedding(ids)
    for block in lm.layers:
        n = add_rms_norm_mx(x, None, block.ssm_norm.weight, eps=block.ssm_norm.eps)[1]
        y, _ = block.ssm.ssd_from_proj(mx_linear(n, quantize_mx(block.ssm.in_proj.weight.detach()), out_dtype=x.dtype))
        x = mx_linear(quantize_mx(y, "e4m3"), quantize_mx(block.ssm.out_proj.weight.detach()), x, block.residual_scale)
        if block.use_mlp:
            m = block.mlp
            n = add_rms_norm_mx(x, None, block.mlp_norm.weight, eps=block.mlp_norm.eps)[1]
            gate_up = mx_linear(n, quantize_mx(torch.cat((m.w_gate.weight, m.w_up.weight)).detach()), out_dtype=x.dtype)
            x = mx_linear(silu_mul_mx(gate_up), quantize_mx(m.w_down.weight.detach()), x, block.residual_scale)
    n = add_rms_norm_mx(x, None, lm.norm.weight, eps=lm.norm.eps)[1]
    return mx_linear(n, quantize_mx(lm.lm_head.weight.detach()), out_dtype=x.dtype)


@torch.no_grad()
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("use_mlp", [True, False])
@pytest.mark.parametrize("batch,seq", [(1, 1), (2, 7), (3, 100)])
def test_model_is_the_operators_one_by_one(batch, seq, use_mlp, dtype):
    lm = small_lm(dtype, use_mlp=use_mlp)
    ids = torch.randint(0, 500, (batch, seq), generator=torch.Generator().manual_seed(1)).cuda()
    plain = lm(ids)["logits"]
    assert lm.quantize_mx() is lm
    got = lm(ids, labels=ids)
    assert same(got["logits"], by_hand(lm, ids)) and not torch.equal(got["logits"], plain)
    if seq > 1:
        torch.testing.assert_close(lm.loss(ids, ids), F.cross_entropy(got["logits"][:, :-1].flatten(0, 1).float(), ids[:, 1:].flatten()))
    assert same(lm.quantize_mx(False)(ids)["logits"], plain)
    assert not any("_mx" in m.__dict__ for m in lm.modules())


@torch.no_grad()
def test_model_quantised_and_not_are_near():
    """Against the same weights' values in the ordinary products: what remains is the rounding of the activations to e4m3, at
    most 2^-4 of each, in the products of a branch (two behind one another, the state's own sums between them), and bf16."""
    lm = small_lm(torch.float32)
    ids = torch.randint(0, 500, (2, 64), generator=torch.Generator().manual_seed(1)).cuda()
    valued = copy.deepcopy(lm)
    for block in valued.layers:
        for lin in (block.ssm.in_proj, block.ssm.out_proj, block.mlp.w_gate, block.mlp.w_up, block.mlp.w_down):
            lin.weight.copy_(quantize_mx(lin.weight).dequantize(torch.float32))
    lm.quantize_mx()
    x = lm.embedding(ids)
    for block, other in zip(lm.layers, valued.layers):
        y, want = block(x), other(x)
        # a branch's relative error is a few times 2^-4 at worst (its own inputs, and what its gates make of them)
        assert ((y - want).norm() / (want - x).norm()).item() < 4 * 2 ** -4
        x = want


@torch.no_grad()
@pytest.mark.parametrize("batch", [1, 3, 20])
def test_generate_quantised(batch):
    lm = small_lm().quantize_mx()
    ids = torch.randint(0, 500, (batch, 11), generator=torch.Generator().manual_seed(1)).cuda()
    runs = []
    for graph in (True, False):
        lm.decode_graph = graph
        runs.append([lm.generate(ids, 20, temperature=0), lm.generate(ids, 20, temperature=0.8, top_k=40, top_p=0.9, generator=torch.Generator("cuda").manual_seed(3)),
                     lm.generate(ids, 20, temperature=1.3, min_p=0.02, generator=torch.Generator("cuda").manual_seed(4)),
                     lm.generate(ids, 20, temperature=0, top_p=0.5), lm.generate(ids, 20, top_k=1, top_p=1.0), lm.generate(ids, 20, temperature=0.7, top_p=0.0)])
    for a, b in zip(*runs):
        assert same(a, b) and a.shape == (batch, 31) and ((a >= 0) & (a < 500)).all() and same(a[:, :11], ids)
    # the ways to ask for the likeliest token
    for a in runs[0][3:]:
        assert same(a, runs[0][0])
    # a decoded token's logits are the forward's, up to the state's roundings: the first token's exactly
    assert same(runs[0][0][:, 11], by_hand(lm, ids)[:, -1].argmax(-1))


@torch.no_grad()
def test_generate_draws_by_sample_tokens():
    lm = small_lm()
    ids = torch.randint(0, 500, (3, 5), generator=torch.Generator().manual_seed(1)).cuda()
    got = lm.generate(ids, 1, temperature=0.9, top_k=30, top_p=0.8, generator=torch.Generator("cuda").manual_seed(7))
    u = torch.rand(3, device="cuda", generator=torch.Generator("cuda").manual_seed(7))
    assert same(got[:, 5], sample_tokens(lm(ids)["logits"][:, -1], u, 0.9, 30, 0.8))
    # rows without a token go on
    lm.norm.weight.fill_(float("nan"))
    got = lm.generate(ids, 3, top_p=0.9)
    assert same(got[:, 5:], torch.full((3, 3), -1, device="cuda"))
    for bad in (dict(top_p=1.5), dict(min_p=-0.1), dict(top_p=0.5, top_k=0), dict(top_p=0.5, temperature=-1.0)):
        with pytest.raises(ValueError):
            lm.generate(ids, 1, **bad)


@torch.no_grad()
def test_copies_follow_the_weights():
    lm = small_lm().quantize_mx()
    ids = torch.randint(0, 500, (2, 9), generator=torch.Generator().manual_seed(1)).cuda()
    old = lm(ids)["logits"]
    lm.layers[0].ssm.in_proj.weight.mul_(1.5)
    changed = lm(ids)["logits"]
    assert same(changed, by_hand(lm, ids)) and not torch.equal(changed, old)
    lm.layers[1].mlp.w_up.weight = torch.nn.Parameter(lm.layers[1].mlp.w_up.weight.flip(0).contiguous())
    assert same(lm(ids)["logits"], by_hand(lm, ids))
    lm.lm_head.weight.data.add_(1.0)
    lm.quantize_mx()  # that left no trace
    assert same(lm(ids)["logits"], by_hand(lm, ids))
    twin = copy.deepcopy(lm)
    twin.layers[0].ssm.out_proj.weight.neg_()
    assert same(twin(ids)["logits"], by_hand(twin, ids)) and same(lm(ids)["logits"], by_hand(lm, ids))


def test_training_is_not_touched_and_hooks_are_refused():
    lm = small_lm(torch.float32)
    ids = torch.randint(0, 500, (2, 9), generator=torch.Generator().manual_seed(1)).cuda()
    grads = []
    for on in (False, True):
        lm.quantize_mx(on)
        lm.zero_grad()
        lm.loss(ids, ids).backward()
        grads.append([p.grad.clone() for p in lm.parameters()])
    assert all(torch.equal(a, b) for a, b in zip(*grads))
    hook = lm.layers[0].mlp.w_up.register_forward_hook(lambda *a: None)
    with torch.no_grad(), pytest.raises(RuntimeError, match="hooks"):
        lm(ids)
    hook.remove()
    biased = small_lm(bias=True)
    with pytest.raises(RuntimeError, match="bias"):
        biased.quantize_mx()
    assert not biased.mx_weights and not biased.layers[0].mx_weights


@torch.no_grad()
def test_copies_are_not_made_in_a_graph():
    lm = small_lm().quantize_mx()
    x = normal((2, 128), 0, torch.bfloat16)
    lm._mx_logits(x)
    want = lm._mx_logits(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = lm._mx_logits(x)
    for i in range(3):
        got.zero_()
        graph.replay()
        assert same(got, want)
    lm.norm.weight.mul_(2.0)
    lm.lm_head.weight.mul_(2.0)
    graph2 = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(graph2):
            lm._mx_logits(x)
    torch.cuda.synchronize()
    assert torch.isfinite(lm._mx_logits(x)).all()


# ---------------------------------------------------------------- graphs, streams, compilation
def serve(x, res, nw, w, w2, u):
    total, q = add_rms_norm_mx(x, res, nw, 0.5)
    h = mx_linear(q, w)
    z = mx_linear(silu_mul_mx(h), w2, out_dtype=torch.float32)
    z2 = mx_linear(h, w2, out_dtype=torch.bfloat16, gated=True)
    tokens, lp = sample_tokens(z, u, 0.8, 40, 0.95, 0.01, return_logprob=True)
    return total, q.data, h, z, z2, tokens, lp, quantize_mx(total).dequantize()


def serve_inputs(rows, seed):
    return (normal((rows, 256), seed, torch.bfloat16), normal((rows, 256), seed + 1, torch.bfloat16), normal((256,), seed + 2, torch.bfloat16),
            quantize_mx(normal((384, 256), seed + 3)), quantize_mx(normal((700, 192), seed + 4)), torch.rand(rows, generator=torch.Generator().manual_seed(seed)).cuda())


@torch.no_grad()
@pytest.mark.parametrize("rows", [3, 300])
def test_two_graphs_and_eager_work_between(rows):
    a, b = serve_inputs(rows, 0), serve_inputs(rows, 10)
    serve(*a)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for args in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(serve(*args))
        graphs.append(g)
    side = torch.cuda.Stream()
    for i in range(4):
        for args in (a, b):
            args[0].copy_(normal(args[0].shape, 100 + i, torch.bfloat16, 1 + i))
            args[5].copy_(torch.rand(rows, generator=torch.Generator().manual_seed(i)))
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        for args, out in zip((a, b), outs):
            for got, want in zip(out, serve(*args)):
                assert same(got, want)


@torch.no_grad()
def test_another_stream():
    args = serve_inputs(40, 0)
    want = serve(*args)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = serve(*args)
    side.synchronize()
    for a, b in zip(got, want):
        assert same(a, b)


def test_backward_captured_while_an_eager_graph_lives():
    x, res, w = (normal(s, i, torch.bfloat16).requires_grad_() for i, s in enumerate([(50, 384), (50, 384), (384,)]))
    dt, dy = normal((50, 384), 5, torch.bfloat16), normal((50, 384), 6, torch.bfloat16)

    def grads():
        total, y = add_rms_norm(x, res, w, 0.5)
        return torch.autograd.grad((total, y), (x, res, w), (dt, dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grads()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = grads()
    for i in range(3):
        with torch.no_grad():
            x.copy_(normal((50, 384), 20 + i, torch.bfloat16))
        want = grads()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert same(a, b)


@torch.no_grad()
def test_compiled():
    torch._dynamo.reset()
    args = serve_inputs(5, 0)
    f = torch.compile(lambda x, res, nw, wd, ws, w2d, w2s, u: serve(x, res, nw, mamba3_amd.MXTensor(wd, ws, (384, 256), "e2m1"),
                                                                    mamba3_amd.MXTensor(w2d, w2s, (700, 192), "e2m1"), u),
                      backend="aot_eager", fullgraph=True)
    x, res, nw, w, w2, u = args
    got = f(x, res, nw, w.data, w.scales, w2.data, w2.scales, u)
    for a, b in zip(got, serve(*args)):
        assert same(a, b)


def test_compiled_gradients():
    torch._dynamo.reset()
    x, res, w = (normal(s, i).requires_grad_() for i, s in enumerate([(50, 384), (50, 384), (384,)]))
    dy = normal((50, 384), 6)

    def f(x, res, w):
        total, y = add_rms_norm(x, res, w, 0.5)
        return (total * 2 + y * dy).sum()

    want = torch.autograd.grad(f(x, res, w), (x, res, w))
    got = torch.autograd.grad(torch.compile(f, backend="aot_eager", fullgraph=True)(x, res, w), (x, res, w))
    for a, b in zip(got, want):
        torch.testing.assert_close(a, b, rtol=0, atol=0)


# ---------------------------------------------------------------- offsets past 32 bits
@torch.no_grad()
def test_many_elements():
    rows, d = 1_100_000, 2048  # 2.25e9 elements
    x = torch.randn(1000, d, device="cuda", dtype=torch.bfloat16).repeat(1100, 1)
    nw = normal((d,), 1, torch.bfloat16)
    total, y = add_rms_norm(x, x, nw, 0.5)
    want = add_rms_norm(x[:1000], x[:1000], nw, 0.5)
    assert same(total[-1000:], want[0]) and same(y[-1000:], want[1])
    del total, y
    q = quantize_mx(x, "e4m3")
    small = quantize_mx(x[:1000], "e4m3")
    assert same(q.data[-1000:], small.data) and same(q.scales[-1000:], small.scales)
    assert same(q.dequantize()[-1000:], small.dequantize())
    w = quantize_mx(normal((5, d), 2))
    assert same(mx_linear(q, w)[-1000:], mx_linear(small, w))
    gated = silu_mul_mx(x)
    small = silu_mul_mx(x[:1000])
    assert same(gated.data[-1000:], small.data) and same(gated.scales[-1000:], small.scales)


@torch.no_grad()
def test_many_results():
    rows, n, k = 70_000, 33_000, 128  # 2.3e9 results
    x, w = normal((1000, k), 0, torch.bfloat16).repeat(70, 1), quantize_mx(normal((n, k), 1))
    got = mx_linear(x, w)
    want = mx_linear(x[:1000].contiguous(), w)
    assert same(got[-1000:], want) and same(got[:1000], want)
    u = torch.rand(1000, generator=torch.Generator().manual_seed(2)).cuda()
    tokens = sample_tokens(got, u.repeat(70), 1.0, 50, 0.9)
    assert same(tokens[-1000:], sample_tokens(want, u, 1.0, 50, 0.9))


# ---------------------------------------------------------------- shapes that a block takes and refuses
@torch.no_grad()
def test_block_shapes_quantised():
    block = small_lm().quantize_mx().layers[0]
    x = normal((3, 1, 128), 0, torch.bfloat16)
    state = block.ssm.allocate_inference_state(3)
    y, after = block.step(x[:, 0], state)
    y3, after3 = block.step(x, state)
    assert y3.shape == x.shape and same(y3[:, 0], y) and all(same(after[k], after3[k]) for k in after)
    for bad in (lambda: block(x[:, 0]), lambda: block.prefill(x[:, 0]), lambda: block(x[:, :0]), lambda: block.step(normal((3, 2, 128), 1, torch.bfloat16), state),
                lambda: block.step(x[:2], state), lambda: block(x[..., :64])):
        with pytest.raises(ValueError):
            bad()
    wide = normal((3, 2, 9, 128), 2, torch.bfloat16)[:, 0]  # rows of a batch that do not follow each other
    assert same(block(wide), block(wide.contiguous()))


@torch.no_grad()
def test_prefill_then_steps_quantised_against_the_forward():
    """The state that a prompt leaves carries the model on: logits of the last tokens, decoded one by one, against those of one
    forward over all. Both round the same activations to 8 bits, but for those that bf16's roundings of the two orders of summing
    set apart: an element that falls to the other side of a tie is off by at most 2^-4 of itself, few do."""
    lm = small_lm(torch.float32).quantize_mx()
    ids = torch.randint(0, 500, (2, 40), generator=torch.Generator().manual_seed(1)).cuda()
    want = lm(ids)["logits"]
    x, states = lm.embedding(ids[:, :32]), []
    for layer in lm.layers:
        x, st = layer.prefill(x)
        states.append(st)
    assert same(lm._mx_logits(x), want[:, :32]) or (lm._mx_logits(x) - want[:, :32]).norm() < 2 ** -4 * want.norm()
    for t in range(32, 40):
        got = lm._next_logits(ids[:, t], states, None)
        assert ((got - want[:, t]).norm() / want[:, t].norm()).item() < 2 ** -4


@pytest.mark.parametrize("kw", [dict(), dict(top_k=5), dict(top_p=0.9), dict(min_p=0.01)])
def test_sample_odd_settings(kw):
    """Temperatures that a division or an exponential would overflow at, and views with steps."""
    z = normal((4, 1000), 0, std=3.0)
    z[:, 17] = 20.0
    u = torch.tensor([0.0, 0.3, 0.6, 0.999]).cuda()
    for t in (1e-320, 1e-45, 1e-30, 1e-6):
        assert same(sample_tokens(z, u, t, **kw), torch.full((4,), 17, device="cuda"))
    for t in (1e30, float("inf")):
        tokens, lp = sample_tokens(z, u, t, return_logprob=True, **kw)
        assert ((tokens >= 0) & (tokens < 1000)).all() and torch.isfinite(lp).all()
        if not kw:  # all masses are alike: the tokens in the order of their logits, ties of the mass or not
            order = z.sort(dim=1, descending=True, stable=True).indices
            assert same(tokens, order.gather(1, (u.double() * 1000).long()[:, None])[:, 0])
    wide = normal((4, 3, 1000), 1)
    assert same(sample_tokens(wide[:, 1], u, **kw), sample_tokens(wide[:, 1].contiguous(), u, **kw))
    assert same(sample_tokens(wide[:, 1], u[1:2].expand(4), **kw), sample_tokens(wide[:, 1], torch.full((4,), 0.3).cuda(), **kw))
    assert same(sample_tokens(wide, u[:, None].expand(4, 3), **kw), sample_tokens(wide.flatten(0, 1), u.repeat_interleave(3), **kw).view(4, 3))


def test_a_captured_graph_follows_the_weights():
    lm = small_lm().quantize_mx()
    x = normal((2, 128), 0, torch.bfloat16)
    with torch.inference_mode():
        first = lm._mx_logits(x).clone()
    with torch.no_grad():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = lm._mx_logits(x)
        graph.replay()
        assert same(got, first)
        lm.lm_head.weight.mul_(3.0)
        want = lm._mx_logits(x)  # makes the copy anew
        graph.replay()
        assert same(got, want) and not torch.equal(got, first)
    with torch.inference_mode():
        lm.lm_head.weight.mul_(0.5)
        want = lm._mx_logits(x).clone()
    with torch.no_grad():
        assert same(lm._mx_logits(x), want)


@torch.no_grad()
def test_compiled_model_runs_its_4_bit_blocks_as_they_are():
    torch._dynamo.reset()
    lm = small_lm().quantize_mx()
    ids = torch.randint(0, 500, (2, 9), generator=torch.Generator().manual_seed(1)).cuda()
    want = lm(ids)["logits"]
    assert same(torch.compile(lm, backend="aot_eager")(ids)["logits"], want)
    torch._dynamo.reset()
