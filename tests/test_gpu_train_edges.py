"""The training operators at the edges of what their documentation allows: saturated and infinite values, a
vocabulary in several pieces, gradients that share memory, modules that do more than their weights say, other
row counts under compilation. Bounds as in test_gpu_train_ops."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import mamba3_amd
from mamba3_amd import _native
from test_gpu_train_ops import DTYPES, HALF, STEP, _lm, hold, mlp_inputs, randn, xent_expected, xent_inputs

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- the gated MLP
def _gates(values, dtype, up=1.0, dy=1.0):
    """One row through an MLP whose hidden unit j has gate values[j] (the sum of its entries) and the given up
    value: (y, dg, du) of the units, read off as gradients of the weights' columns that x's 1 meets."""
    n = len(values)
    terms = torch.tensor(values, device="cuda").to(dtype).view(n, -1)
    x = torch.zeros(1, 8, device="cuda", dtype=dtype)
    x[0, :terms.shape[1]] = 1.0
    wg = torch.zeros(n, 8, device="cuda", dtype=dtype)
    wg[:, :terms.shape[1]] = terms
    wu = torch.zeros(n, 8, device="cuda", dtype=dtype)
    wu[:, 0] = up
    wd = torch.eye(8, n, device="cuda", dtype=dtype)
    wg.requires_grad_(), wu.requires_grad_()
    y = mamba3_amd.swiglu_mlp(x, wg, wu, wd)
    dwg, dwu = torch.autograd.grad(y, [wg, wu], torch.full_like(y, dy))
    return wg.detach().double().sum(1), dwg[:, 0].double(), dwu[:, 0].double()


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp32"])
@pytest.mark.parametrize("up", [1.0, 3e37, -3e37])
def test_mlp_saturated_gates_meet_large_gradients(dtype, up):
    """Far-out gates under a gradient of several units: silu and its slope are 0 or as good as 0 there, and their
    products with large factors 0 as well, not infinity times zero."""
    gates = [-3e38, -1e38, -1e30, -200.0, 200.0, 1e4, 1e30, 1e37]
    g, dg, du = _gates([[v] for v in gates], dtype, up, dy=8.0)
    u = torch.tensor(up).to(dtype).double().item()
    flat = g < -100.0
    slope, silu = torch.where(flat, 0.0, 1.0).double(), torch.where(flat, 0.0, g)
    assert torch.allclose(du, 8.0 * silu, rtol=2 * HALF[dtype] + 8 * STEP, atol=1e-30), du
    assert torch.allclose(dg, 8.0 * u * slope, rtol=2 * HALF[dtype] + 8 * STEP, atol=1e-30), dg


def test_mlp_kept_gates_are_rounded_to_the_nearest():
    """What the backward reads of a gate in bf16 has 16 significant bits: half a step of those, 2^-16 in [1, 2), is
    how far it may be off. Near the zero of silu' (g = -1.2784645) a gate's error is all that is left of dg: gates
    there whose last bits, 2^-15 and below, are just under a whole step."""
    root, a, step = 1.2784645427610738, 1.2734375, 2.0 ** -15
    base = math.floor((root - a) / step)
    gates = [[-a, -(base + i) * step, -f * step] for i in (-4, -1, 0, 3) for f in (0.96875, 0.5625)]
    g, dg, _ = _gates(gates, torch.bfloat16)
    assert ((g + root).abs() < 2.0 ** -12).all()
    s = torch.sigmoid(g)
    want = s * (1 + g * (1 - s))
    # |silu''| <= 0.2195 around here; the slope's own fp32 steps; dg and its gradient are rounded to bf16
    bound = 0.2195 * 2.0 ** -16 + (g.abs() + 4) * 2.0 ** -21 * s * (1 + g.abs()) + 2 * HALF[torch.bfloat16] * want.abs()
    assert ((dg - want).abs() <= bound).all(), ((dg - want).abs() / bound).max().item()


@pytest.mark.parametrize("rows", [8, 60])
def test_mlp_fp32_rounding_of_a_long_sum(rows):
    """fp32 products of few rows sum every 512 k apart. With random terms of size s the j-th partial sum is about
    sqrt(j) s, and its rounding at most 2^-24 of it, evenly spread: a variance of (2^-23)^2 / 12 j s^2. Over blocks of n of
    K terms that is (2^-23)^2 n / 24 of the sum's own variance K s^2, and as much for the K / n sums of blocks. (One chain
    over all K would be off by sqrt(K / 24) 2^-23.) The up projection is seen through a gate of 32, whose silu is 32,
    and a down projection that copies."""
    d, ff, n = 16384, 64, 512
    x = randn(rows, d, dtype=torch.float32, seed=1)
    up = randn(ff, d, dtype=torch.float32, seed=2)
    gate = torch.zeros(ff, d, device="cuda")
    x[:, 0], gate[:, 0], up[:, 0] = 1.0, 32.0, 0.0
    y = mamba3_amd.swiglu_mlp(x, gate, up, torch.eye(d, ff, device="cuda"))[:, :ff].double() / 32
    want = x.double() @ up.double().t()
    off = (y - want).square().mean().sqrt() / want.square().mean().sqrt()
    assert off <= STEP * math.sqrt((n + d / n) / 24), off.item() / STEP


# ---------------------------------------------------------------- the linear cross entropy
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp32"])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_xent_ignored_rows_add_nothing_to_a_weight_that_is_not_finite(dtype, value):
    """dweight is a sum over the rows that count: without any it is zero, whatever the weight holds."""
    hidden, weight, _ = xent_inputs(40, 48, 300, dtype)
    weight[7, 3], weight[290] = value, value
    target = torch.full((40,), -100, device="cuda")
    for reduction in ("mean", "sum", "none"):
        h, w = hidden.detach().requires_grad_(), weight.detach().requires_grad_()
        loss = mamba3_amd.linear_cross_entropy(h, w, target, reduction=reduction)
        (dw,) = torch.autograd.grad(loss.sum(), [w])
        assert not dw.any(), reduction
        if reduction != "mean":
            assert not loss.any()


@pytest.mark.parametrize("wanted", ["both", "hidden", "weight"])
@pytest.mark.parametrize("rows,d,vocab,dtype,reduction", [
    (4096, 100, 40000, torch.bfloat16, "none"), (4096, 64, 40000, torch.bfloat16, "sum"),
    (4096, 33, 20000, torch.float32, "none"), (4100, 64, 20011, torch.float32, "mean")])
def test_xent_pieces_of_the_vocabulary(rows, d, vocab, dtype, reduction, wanted):
    """The backward's loop over pieces: types, reductions, widths that 16 bytes do not divide, one gradient alone."""
    print(rows, d, vocab, dtype, reduction, wanted, flush=True)
    n = ctypes.c_size_t(0)
    assert _native.lib().m3_linear_xent_bwd_workspace_size(rows, d, vocab, _native.dtype_code(dtype), 0, 0, ctypes.byref(n)) == 0
    assert n.value < rows * vocab * dtype.itemsize  # more than one piece
    hidden, weight, target = xent_inputs(rows, d, vocab, dtype)
    target[0] = vocab - 1
    hidden.requires_grad_(wanted != "weight")
    weight.requires_grad_(wanted != "hidden")
    loss = mamba3_amd.linear_cross_entropy(hidden, weight, target, reduction=reduction)
    grad = randn(rows, dtype=torch.float32, seed=5) if reduction == "none" else torch.tensor(1.5, device="cuda")
    leaves = [t for t in (hidden, weight) if t.requires_grad]
    got = dict(zip([k for k, t in (("dhidden", hidden), ("dweight", weight)) if t.requires_grad], torch.autograd.grad(loss, leaves, grad)))
    want = dict(zip(("loss", "dhidden", "dweight"), xent_expected(hidden, weight, target, reduction, grad, dtype)))
    for name, g in {"loss": loss, **got}.items():
        hold(name, g, want[name])


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp32"])
def test_xent_small_losses_of_large_logits(dtype):
    """Logits of thousands that lie a few units apart: the loss is their difference, log sum exp(z - top) + (top -
    z_target), and no number as large as the logits is rounded on the way."""
    top = 4096.0
    steps = [0.0, 2.0, 3.0, 5.0, 8.0, 16.0]
    hidden = torch.full((len(steps), 8), 0.0, device="cuda", dtype=dtype)
    hidden[:, 0], hidden[:, 1] = 64.0, 1.0
    weight = torch.zeros(len(steps) + 50, 8, device="cuda", dtype=dtype)
    weight[:len(steps), 0] = top / 64
    weight[:len(steps), 1] = -torch.tensor(steps, device="cuda").to(dtype)
    target = torch.arange(len(steps), device="cuda")
    loss = mamba3_amd.linear_cross_entropy(hidden, weight, target, reduction="none").double()
    z = top - torch.tensor(steps, device="cuda").double()
    log_sum = torch.log(torch.exp(z - top).sum())
    want = log_sum + (top - z)
    # the exponentials' and the logarithm's steps, one addition
    assert ((loss - want).abs() <= (16 + 4) * 2.0 ** -22 + 4 * STEP * want).all(), (loss - want).abs().max().item()


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp32"])
@pytest.mark.parametrize("vocab", [64, 700, 1029])
def test_xent_logits_at_the_types_lowest_value(dtype, vocab):
    """Whole tiles of columns, and whole rows, at the lowest finite value: they take no part beside others, and are
    as good as one another alone."""
    low = torch.finfo(dtype).min
    hidden = torch.zeros(4, 8, device="cuda", dtype=dtype)
    hidden[0, 0], hidden[1, 1], hidden[2, 2], hidden[3, 3] = 1.0, 1.0, 1.0, 1.0
    weight = torch.zeros(vocab, 8, device="cuda", dtype=dtype)
    weight[:, 0] = low                                # row 0: nothing but the lowest
    weight[: vocab - 20, 1] = low                     # row 1: all columns but the last
    weight[30:, 2] = low                              # row 2: all columns but the first
    weight[::3, 3] = low
    weight[:, 4] = torch.linspace(-2, 2, vocab).to(dtype)
    hidden[1:, 4] = 1.0
    target = torch.tensor([5, vocab - 3, 7, 10], device="cuda")
    loss = mamba3_amd.linear_cross_entropy(hidden, weight, target, reduction="none")
    z = hidden.detach().double() @ weight.detach().double().t()
    want = torch.nn.functional.cross_entropy(z, target, reduction="none")
    assert ((loss.double() - want).abs() <= 64 * STEP * (1 + want)).all(), (loss, want)
    # (the gradient takes exp(z - lse) from an lse in fp32: row 0's is no more than its maximum)
    h, w = hidden.detach()[1:].requires_grad_(), weight.detach().requires_grad_()
    dw = torch.autograd.grad(mamba3_amd.linear_cross_entropy(h, w, target[1:], reduction="sum"), w)[0].double()
    dz = torch.softmax(z[1:], 1)
    dz[torch.arange(3, device="cuda"), target[1:]] -= 1
    size = dz.abs().t() @ h.detach().double().abs()
    assert ((dw - dz.t() @ h.detach().double()).abs() <= size * (2 * HALF[dtype] + 64 * STEP) + STEP).all()


# ---------------------------------------------------------------- modules
class _Doubled(torch.nn.Linear):
    def forward(self, x):
        return 2 * super().forward(x)


def _mlp_of(lm):
    return lm.layers[0].mlp


@pytest.mark.parametrize("name", ["w_gate", "w_up", "w_down", "lm_head"])
@pytest.mark.parametrize("how", ["hook", "pre_hook", "subclass", "forward", "global"])
def test_modules_with_more_than_a_weight_are_called(name, how):
    """A projection with hooks or a forward of its own: fuse_mlp and loss give what the path without them gives."""
    ids = torch.randint(300, (2, 20), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    # (without checkpointing the block reads w_down's weight for its residual)
    lm = _lm(torch.float32, tie_weights=False, gradient_checkpointing=name == "w_down").train()
    owner = lm if name == "lm_head" else _mlp_of(lm)
    lin, undo = getattr(owner, name), None
    if how == "hook":
        lin.register_forward_hook(lambda m, args, out: 2 * out)
    elif how == "pre_hook":
        lin.register_forward_pre_hook(lambda m, args: (2 * args[0],))
    elif how == "subclass":
        twice = _Doubled(lin.in_features, lin.out_features, bias=False).cuda()
        twice.load_state_dict(lin.state_dict())
        setattr(owner, name, twice)
    elif how == "forward":
        plain = lin.forward
        lin.forward = lambda x: 2 * plain(x)
    else:
        undo = torch.nn.modules.module.register_module_forward_hook(lambda m, args, out: 2 * out if m is lin else None)
    try:
        want = lm(ids, ids)["loss"]
        want_g = torch.autograd.grad(want, lm.embedding.weight)[0]
        got = lm.fuse_mlp().loss(ids, ids)
        got_g = torch.autograd.grad(got, lm.embedding.weight)[0]
    finally:
        if undo is not None:
            undo.remove()
    assert abs(got.item() - want.item()) <= 1e-5 * abs(want.item())
    assert (got_g - want_g).norm() <= 1e-4 * want_g.norm()


def test_hooks_of_the_mlp_itself_are_called():
    ids = torch.randint(300, (2, 20), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    lm = _lm(torch.float32, gradient_checkpointing=True).train()
    _mlp_of(lm).register_forward_hook(lambda m, args, out: 2 * out)
    want = lm(ids, ids)["loss"].item()
    assert abs(lm.fuse_mlp().loss(ids, ids).item() - want) <= 1e-5 * want


def test_loss_of_a_head_with_a_bias():
    ids = torch.randint(300, (2, 20), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    lm = _lm(torch.float32, tie_weights=False)
    head = torch.nn.Linear(128, 300).cuda()
    lm.lm_head = head
    labels = ids.clone()
    labels[0, 5:9] = 7
    want = lm(ids, ids)["loss"]
    assert abs(lm.loss(ids, ids).item() - want.item()) <= 1e-5 * want.item()
    want = lm(ids, torch.where(labels == 7, -100, labels))["loss"]
    assert abs(lm.loss(ids, labels, ignore_index=7).item() - want.item()) <= 1e-5 * want.item()


def test_language_model_compiles_with_its_fused_mlp():
    ids = torch.randint(300, (2, 20), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    lm = _lm(torch.bfloat16).train().fuse_mlp()
    want = torch.autograd.grad(lm.loss(ids, ids), lm.embedding.weight)[0]
    got = torch.autograd.grad(torch.compile(lm.loss, fullgraph=True)(ids, ids), lm.embedding.weight)[0]
    # the compiler may keep what eager code rounds between operators
    assert (got.float() - want.float()).norm() <= 16 * HALF[torch.bfloat16] * want.float().norm()


# ---------------------------------------------------------------- clipping
def _with_grads(*grads):
    out = []
    for g in grads:
        p = torch.nn.Parameter(torch.empty(g.shape, device="cuda", dtype=g.dtype))
        p.grad = g
        out.append(p)
    return out


def test_clip_refuses_strided_gradients_that_share_memory():
    base = randn(64, 40, dtype=torch.float32, seed=3)
    kept = base.clone()
    shared = [
        (base[:, :20], base[:, 19:]),                       # columns that meet in one
        (base[::2], base[:3]),                              # every second row, and the first rows
        (base.t(), base[10:11]),                            # all of it transposed, and a row
        (base.flatten()[::3], base.flatten()[1::2]),        # different steps through the same numbers
        (base.as_strided((10, 10), (5, 1)),),               # one that meets itself
        (base[:, 3].expand(4, 64).t(),),
    ]
    for grads in shared:
        with pytest.raises(ValueError, match="overlap|share memory"):
            mamba3_amd.clip_grad_norm_(_with_grads(*grads), 1.0)
    assert torch.equal(base, kept)


def test_clip_takes_interleaved_gradients():
    """Views of one buffer that lie between one another's elements: every element counts, and is scaled, once."""
    for cut in (lambda b: (b[:, :13], b[:, 13:14], b[:, 14:]), lambda b: (b[::2], b[1::2]),
                lambda b: (b.flatten()[::3], b.flatten()[1::3], b.flatten()[2::3]),
                lambda b: (b[:32].t(), b[32:]), lambda b: (b.flatten()[::4], b.flatten()[2::4], b.flatten()[1::2])):
        base = randn(64, 40, dtype=torch.float32, seed=3)
        want = base.double()
        norm = want.norm().item()
        got = mamba3_amd.clip_grad_norm_(_with_grads(*cut(base)), 0.5).item()
        assert abs(got - norm) <= STEP * norm
        want = want * (0.5 / (norm + 1e-6))
        assert ((base.double() - want).abs() <= want.abs() * (HALF[torch.float32] + 2 * STEP)).all()


# ---------------------------------------------------------------- compilation
def test_compiled_once_for_all_row_counts():
    """With rows marked dynamic one compilation serves every number of rows, forward and backward."""
    t = mlp_inputs(64, 128, 320, torch.bfloat16)
    _, head, _ = xent_inputs(64, 128, 1000, torch.bfloat16)
    leaves = [t[k].requires_grad_() for k in ("w_gate", "w_up", "w_down")] + [head.requires_grad_()]
    from torch._dynamo.backends.common import aot_autograd
    compiled = []

    def backend(graph, inputs):
        compiled.append(len(inputs))
        return graph.forward

    def f(x, target):
        return mamba3_amd.linear_cross_entropy(mamba3_amd.swiglu_mlp(x, *leaves[:3], residual=x), head, target)

    torch._dynamo.reset()
    step = torch.compile(f, fullgraph=True, backend=aot_autograd(fw_compiler=backend))
    for rows in (64, 3, 17, 40, 100, 257, 300, 31, 999, 1000, 8):
        x = randn(rows, 128, dtype=torch.bfloat16, seed=rows)
        target = torch.arange(rows, device="cuda")
        torch._dynamo.mark_dynamic(x, 0)
        torch._dynamo.mark_dynamic(target, 0)
        want = torch.autograd.grad(f(x, target), leaves)
        got = torch.autograd.grad(step(x, target), leaves)
        assert all(torch.equal(a, b) for a, b in zip(want, got)), rows
    assert len(compiled) == 2  # a forward and a backward graph


# ---------------------------------------------------------------- devices
def test_few_rows_run_on_their_own_device(monkeypatch):
    """The decode kernels that take few rows run inside ops.on_device, as the tiles do."""
    from mamba3_amd import ops
    t = mlp_inputs(4, 128, 320, torch.bfloat16)
    inside, seen = [], []
    real = ops.on_device

    class Watched:
        def __init__(self, x):
            self.real = real(x)

        def __enter__(self):
            inside.append(1)
            return self.real.__enter__()

        def __exit__(self, *a):
            inside.pop()
            return self.real.__exit__(*a)

    monkeypatch.setattr(ops, "on_device", Watched)
    for name in ("small_swiglu_fast", "small_linear_fast"):
        fn = getattr(ops, name)
        monkeypatch.setattr(ops, name, lambda *a, fn=fn: (seen.append(len(inside)), fn(*a))[1])
    with torch.no_grad():
        mamba3_amd.swiglu_mlp(**t)
    assert seen == [1, 1]


# ---------------------------------------------------------------- graphs
@pytest.mark.parametrize("rows,d,vocab,dtype", [(16, 256, 50021, torch.float32), (4096, 100, 40000, torch.bfloat16)])
def test_captured_loss_replays(rows, d, vocab, dtype):
    """Two captured losses with their gradients, one after the other, between eager ones: few rows (dh and dW in launches
    of their own, dh in parts) and several pieces of the vocabulary (sums kept from piece to piece)."""
    print(rows, d, vocab, dtype, flush=True)

    def run(h, w, t):
        loss = mamba3_amd.linear_cross_entropy(h, w, t)
        return [loss.detach(), *torch.autograd.grad(loss, [h, w])]

    inputs = {s: xent_inputs(rows, d, vocab, dtype, seed=s) for s in (0, 10, 20)}
    for h, w, t in inputs.values():
        t[0] = 5
    eager = {s: run(h.clone().requires_grad_(), w.clone().requires_grad_(), t) for s, (h, w, t) in inputs.items()}
    graphs = []
    for _ in range(2):
        h, w, t = (v.clone() for v in inputs[0])
        h.requires_grad_(), w.requires_grad_()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(h, w, t)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(h, w, t)
        graphs.append((graph, (h, w, t), out))
    for seeds in ((10, 20), (20, 0), (0, 10)):
        for (graph, own, out), s in zip(graphs, seeds):
            for a, b in zip(own, inputs[s]):
                with torch.no_grad():
                    a.copy_(b)
            graph.replay()
        torch.cuda.synchronize()
        for (graph, own, out), s in zip(graphs, seeds):
            assert all(torch.equal(a, b) for a, b in zip(out, eager[s]))
        run(*(v.clone().requires_grad_() if v.is_floating_point() else v for v in inputs[0]))
