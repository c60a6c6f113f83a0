"""The training operators on the GPU against their definitions in 64 bits.

Tolerances are not chosen but carried along: a `Num` holds a value in fp64 and a bound on how far a
kernel's intermediate may be from it, and each step adds its own: a rounding to a type half a step
(2^-8 bf16, 2^-24 fp32, relative), a product over k terms k + 2 additions of at most one fp32 step
(2^-23) of the terms' magnitudes, an exponential of x a relative (|x| + 4) 2^-22 (its argument's
rounding and the instruction's own step). Outputs are held to their bound element by element."""

from __future__ import annotations

import math

import pytest
import torch

import mamba3_amd
from mamba3_amd import _native

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
STEP = 2.0 ** -23
TINY = 1e-30  # products below the normal range of the types
DTYPES = [torch.bfloat16, torch.float32]


class Num:
    def __init__(self, v, e=None):
        self.v = v.detach().double()
        self.e = torch.zeros_like(self.v) if e is None else e

    @property
    def top(self):
        return self.v.abs() + self.e

    def t(self):
        return Num(self.v.t(), self.e.t())

    def rounded(self, dtype):
        return Num(self.v, self.e + HALF[dtype] * self.top)

    def rel(self, r):
        return Num(self.v, self.e + r * self.top)

    def __mul__(self, o):
        if not isinstance(o, Num):
            return Num(self.v * o, self.e * abs(o) + STEP * self.top * abs(o))
        return Num(self.v * o.v, self.top * o.top - (self.v * o.v).abs() + STEP * self.top * o.top)

    def __add__(self, o):
        return Num(self.v + o.v, self.e + o.e + STEP * (self.top + o.top))

    def dot(self, o):
        """self o^T: rows of k times rows of k."""
        k = self.v.shape[1]
        size = self.top @ o.top.t()
        return Num(self.v @ o.v.t(), size - self.v.abs() @ o.v.abs().t() + (k + 2) * STEP * size)


def sigmoid(g):
    s = torch.sigmoid(g.v)
    return Num(s, 0.25 * g.e + (g.top + 4) * 2.0 ** -22 * s)


def hold(name, got, want, dtype=None):
    got = got.detach().double()
    assert got.shape == want.v.shape, name
    off = (got - want.v).abs()
    bad = ~(off <= want.e * (1 + 1e-6) + TINY)
    worst = (off / (want.e + TINY)).max().item() if off.numel() else 0.0
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} past the bound, {worst:.3g} times at worst"


def randn(*shape, dtype, seed, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


# ---------------------------------------------------------------- the gated MLP
def mlp_inputs(rows, d, ff, dtype, seed=0, residual=True):
    w = 1.0 / math.sqrt(d)
    return dict(x=randn(rows, d, dtype=dtype, seed=seed), w_gate=randn(ff, d, dtype=dtype, seed=seed + 1, std=w),
                w_up=randn(ff, d, dtype=dtype, seed=seed + 2, std=w),
                w_down=randn(d, ff, dtype=dtype, seed=seed + 3, std=1.0 / math.sqrt(ff)),
                residual=randn(rows, d, dtype=dtype, seed=seed + 4) if residual else None)


def mlp_expected(t, scale, dy, dtype):
    """{output: Num} of swiglu_mlp on 2-D inputs."""
    x, wg, wu, wd = (Num(t[k]) for k in ("x", "w_gate", "w_up", "w_down"))
    g, u = x.dot(wg), x.dot(wu)
    s = sigmoid(g)
    h = (g * s * u).rounded(dtype)
    y = h.dot(wd) * scale
    if t.get("residual") is not None:
        y = y + Num(t["residual"])
    out = {"y": y.rounded(dtype)}
    if dy is None:
        return out
    # kept for the backward: 16 significant bits (bf16), all of them (fp32)
    if dtype == torch.bfloat16:
        g, u = g.rel(2.0 ** -15), u.rel(2.0 ** -15)
    s = sigmoid(g)
    one = torch.ones_like(g.v)
    # silu' = s (1 + g (1 - s)); |silu''| <= 1/2
    slope = Num(s.v * (1 + g.v * (1 - s.v)), 0.5 * g.e + (g.top + 4) * 2.0 ** -21 * s.v * (1 + g.top))
    dyn = Num(dy)
    dh = dyn.dot(wd.t()) * scale
    dg = (dh * u * slope).rounded(dtype)
    du = (dh * g * s).rounded(dtype)
    out["x"] = (dg.dot(wg.t()) + du.dot(wu.t())).rounded(dtype)
    out["w_gate"] = dg.t().dot(x.t()).rounded(dtype)
    out["w_up"] = du.t().dot(x.t()).rounded(dtype)
    out["w_down"] = (dyn.t().dot(h.t()) * scale).rounded(dtype)
    out["residual"] = Num(dy)
    return out


MLP_SHAPES = [
    (1, 64, 128), (1, 1, 1), (2, 8, 8), (3, 100, 77), (9, 64, 192), (24, 256, 704), (65, 130, 67), (130, 96, 200),
    (257, 264, 136), (300, 513, 1025), (512, 768, 2112), (1000, 500, 1363), (2500, 72, 4100),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp32"])
@pytest.mark.parametrize("rows,d,ff", MLP_SHAPES)
def test_mlp_forward_and_gradients(rows, d, ff, dtype):
    print(rows, d, ff, dtype, flush=True)
    t = mlp_inputs(rows, d, ff, dtype, residual=rows % 2 == 0)
    dy = randn(rows, d, dtype=dtype, seed=9)
    scale = 0.375
    leaves = {k: v.requires_grad_() for k, v in t.items() if v is not None}
    y = mamba3_amd.swiglu_mlp(**t, scale=scale)
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))
    want = mlp_expected(t, scale, dy, dtype)
    assert y.dtype == dtype
    hold("y", y, want["y"])
    for k in leaves:
        assert grads[k].dtype == dtype and grads[k].shape == leaves[k].shape
        hold(k, grads[k], want[k])


@pytest.mark.parametrize("rows,d,ff", [(4096, 768, 2112), (2048, 2048, 5504), (16384, 256, 704)])
def test_mlp_large_tiles(rows, d, ff):
    """The 256 x 256 tiles, products split over their inner length, and rows of whole tiles."""
    print(rows, d, ff, flush=True)
    dtype = torch.bfloat16
    t = mlp_inputs(rows, d, ff, dtype)
    dy = randn(rows, d, dtype=dtype, seed=9)
    leaves = {k: v.requires_grad_() for k, v in t.items()}
    y = mamba3_amd.swiglu_mlp(**t, scale=0.5)
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))
    want = mlp_expected(t, 0.5, dy, dtype)
    hold("y", y, want["y"])
    for k in leaves:
        hold(k, grads[k], want[k])


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp32"])
@pytest.mark.parametrize("rows", [1, 5, 8, 9, 40])
def test_mlp_without_gradients(rows, dtype):
    """Serving: at most 8 bf16 rows run on the decode kernels, others on the tiles."""
    t = mlp_inputs(rows, 128, 320, dtype)
    with torch.no_grad():
        y = mamba3_amd.swiglu_mlp(**t, scale=0.25)
        alone = mamba3_amd.swiglu_mlp(t["x"], t["w_gate"], t["w_up"], t["w_down"])
        scaled = mamba3_amd.swiglu_mlp(t["x"], t["w_gate"], t["w_up"], t["w_down"], scale=0.25)
    hold("y", y, mlp_expected(t, 0.25, None, dtype)["y"])
    t["residual"] = None
    hold("no residual", alone, mlp_expected(t, 1.0, None, dtype)["y"])
    hold("no residual, scaled", scaled, mlp_expected(t, 0.25, None, dtype)["y"])


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp32"])
def test_mlp_strides_and_alignment(dtype):
    """Sliced, transposed and misaligned inputs, a transposed output gradient: values as for copies."""
    rows, d, ff = 37, 72, 104
    t = mlp_inputs(rows, d, ff, dtype)
    dy = randn(rows, d, dtype=dtype, seed=9)

    def odd(v, k):
        if k % 3 == 0:  # every second column of a wider tensor
            w = torch.zeros(v.shape[0], 2 * v.shape[1], device="cuda", dtype=dtype)
            w[:, ::2] = v
            return w[:, ::2]
        if k % 3 == 1:  # transposed storage
            return v.t().contiguous().t()
        w = torch.zeros(v.numel() + 1, device="cuda", dtype=dtype)  # one element off alignment
        w[1:] = v.reshape(-1)
        return w[1:].view(v.shape)

    def run(t, dy):
        leaves = [v.detach().requires_grad_() for v in t.values()]
        y = mamba3_amd.swiglu_mlp(*leaves, scale=0.5)
        return [y, *torch.autograd.grad(y, leaves, dy)]

    base = run(t, dy)
    for shift in range(3):
        got = run({k: odd(v, i + shift) for i, (k, v) in enumerate(t.items())}, odd(dy, shift))
        for a, b in zip(base, got):
            assert torch.equal(a, b)


def test_mlp_batch_dimensions_and_frozen_weights():
    t = mlp_inputs(30, 64, 96, torch.bfloat16)
    dy = randn(30, 64, dtype=torch.bfloat16, seed=9)
    want = mlp_expected(t, 1.0, dy, torch.bfloat16)
    shaped = {k: v.view(2, 3, 5, 64) if k in ("x", "residual") else v for k, v in t.items()}
    for trained in (["x"], ["w_up"], ["w_gate"], ["w_down"], ["residual"], ["w_down", "w_gate"], ["x", "w_up"]):
        leaves = {k: v.detach().clone().requires_grad_(k in trained) for k, v in shaped.items()}
        y = mamba3_amd.swiglu_mlp(**leaves)
        assert y.shape == (2, 3, 5, 64)
        y.backward(dy.view(y.shape))
        for k, v in leaves.items():
            assert (v.grad is not None) == (k in trained)
            if k in trained:
                hold(k, v.grad.reshape(t[k].shape), want[k])


def test_mlp_no_rows():
    t = mlp_inputs(4, 16, 24, torch.float32)
    x = torch.empty(0, 16, device="cuda", requires_grad=True)
    w = t["w_up"].requires_grad_()
    y = mamba3_amd.swiglu_mlp(x, t["w_gate"], w, t["w_down"], residual=x)
    y.sum().backward()
    assert y.shape == (0, 16) and x.grad.shape == (0, 16) and not w.grad.any()


def test_mlp_extreme_gates():
    """Gates far out saturate without overflow: silu(g) -> g or 0, its slope -> 1 or 0."""
    for dtype in DTYPES:
        x = torch.tensor([[1.0] + [0.0] * 7], device="cuda", dtype=dtype).requires_grad_()
        gates = torch.tensor([-3e38, -1e4, -100.0, 0.0, 100.0, 1e4, 1e30, -0.0], device="cuda")
        wg = torch.zeros(8, 8, device="cuda", dtype=dtype)
        wg[:, 0] = gates.to(dtype)
        wu = torch.zeros(8, 8, device="cuda", dtype=dtype)
        wu[:, 0] = 0.5
        wd = torch.eye(8, device="cuda", dtype=dtype)
        y = mamba3_amd.swiglu_mlp(x, wg, wu, wd)
        (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
        g = wg[:, 0].double()
        want = torch.where(g < -90, torch.zeros_like(g), torch.nn.functional.silu(g) * 0.5)
        assert torch.isfinite(y).all() and torch.isfinite(dx).all()
        assert torch.allclose(y[0].double(), want, rtol=2 * HALF[dtype] + 1e-6, atol=1e-30)


def test_mlp_nan_and_inf_reach_their_own_rows_only():
    t = mlp_inputs(20, 64, 96, torch.bfloat16)
    clean = mamba3_amd.swiglu_mlp(**t)
    t["x"][3, 5] = math.nan
    t["x"][7, 0] = math.inf
    y = mamba3_amd.swiglu_mlp(**t)
    rows = [i for i in range(20) if i not in (3, 7)]
    assert torch.equal(y[rows], clean[rows]) and torch.isnan(y[3]).all() and not torch.isfinite(y[7]).all()


def test_mlp_gradient_against_differences():
    """fp32 gradients along random directions against central differences of the definition in
    64 bits (step 1e-5: truncation below 1e-9 of these smooth values)."""
    dtype = torch.float32
    t = mlp_inputs(6, 24, 40, dtype)
    dy = randn(6, 24, dtype=dtype, seed=9)
    leaves = {k: v.requires_grad_() for k, v in t.items()}
    grads = dict(zip(leaves, torch.autograd.grad(mamba3_amd.swiglu_mlp(**t, scale=0.7), list(leaves.values()), dy)))
    want = mlp_expected(t, 0.7, dy, dtype)

    def f(v):
        g, u = v["x"] @ v["w_gate"].t(), v["x"] @ v["w_up"].t()
        return ((v["residual"] + 0.7 * (g / (1 + torch.exp(-g)) * u) @ v["w_down"].t()) * dy.double()).sum().item()

    for k in leaves:
        way = randn(*t[k].shape, dtype=torch.float32, seed=21).double()
        base = {n: v.detach().double() for n, v in t.items()}
        up, down = dict(base), dict(base)
        up[k], down[k] = base[k] + 1e-5 * way, base[k] - 1e-5 * way
        slope = (f(up) - f(down)) / 2e-5
        allowed = (want[k].e * way.abs()).sum().item() + 1e-8 * (1 + abs(slope))
        assert abs((grads[k].double() * way).sum().item() - slope) <= allowed, k


# ---------------------------------------------------------------- the linear cross entropy
def xent_inputs(rows, d, vocab, dtype, seed=0, ignored=0.2):
    hidden = randn(rows, d, dtype=dtype, seed=seed)
    weight = randn(vocab, d, dtype=dtype, seed=seed + 1, std=3.0 / math.sqrt(d))
    g = torch.Generator(device="cuda").manual_seed(seed + 2)
    target = torch.randint(vocab, (rows,), generator=g, device="cuda")
    skip = torch.rand(rows, generator=g, device="cuda") < ignored
    return hidden, weight, torch.where(skip, -100, target)


def xent_expected(hidden, weight, target, reduction, grad, dtype, ignore=-100):
    rows, vocab = hidden.shape[0], weight.shape[0]
    h, w = Num(hidden), Num(weight)
    live = target != ignore
    at = torch.where(live, target, 0)[:, None]
    z = h.dot(w)
    lse = torch.logsumexp(z.v, 1, keepdim=True)
    far = (z.v.amax(1, keepdim=True) - z.v).clamp(max=40.0)  # terms further out do not matter
    share = torch.exp(z.v - lse)
    # the terms' errors weighted by their share, and the additions of the sum
    e_lse = (share * (z.e + (far + 4) * 2.0 ** -22)).sum(1, keepdim=True) * 1.01 + (64 + vocab / 256) * STEP + lse.abs() * STEP * 2
    pick = Num(z.v.gather(1, at), z.e.gather(1, at))
    row = Num((lse - pick.v)[:, 0], (e_lse + pick.e)[:, 0] + STEP * (lse.abs() + pick.v.abs())[:, 0])
    row = Num(torch.where(live, row.v, 0.0), torch.where(live, row.e, 0.0))
    n = live.sum()
    if reduction == "none":
        loss = row
        gl = torch.as_tensor(grad, device="cuda").double().expand(rows)
    else:
        div = n.double() if reduction == "mean" else 1.0
        loss = Num(row.v.sum() / div, (row.e.sum() + STEP * row.top.sum()) / div)
        gl = (torch.as_tensor(grad, device="cuda").double() / div).expand(rows)
    p = torch.exp(z.v - lse)
    e_p = p * torch.expm1(z.e + e_lse + ((z.v - lse).abs() + 4) * 2.0 ** -22)
    one = torch.zeros_like(p).scatter_(1, at, 1.0)
    dz = Num(p - one, e_p + STEP)
    scale = torch.where(live, gl, 0.0)[:, None]
    dz = Num(dz.v * scale, dz.e * scale.abs() + 2 * STEP * dz.top * scale.abs()).rounded(dtype)
    clean = Num(torch.where(live[:, None], h.v, 0.0))
    return loss, dz.dot(w.t()).rounded(dtype), dz.t().dot(clean.t()).rounded(dtype)


XENT_SHAPES = [(1, 8, 1), (1, 64, 300), (2, 1, 5), (5, 33, 7), (64, 64, 256), (65, 72, 1000), (130, 100, 513),
               (300, 256, 4099), (777, 768, 2000), (2050, 64, 259)]


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp32"])
@pytest.mark.parametrize("rows,d,vocab", XENT_SHAPES)
def test_xent_loss_and_gradients(rows, d, vocab, dtype):
    for reduction in ("mean", "sum", "none"):
        print(rows, d, vocab, dtype, reduction, flush=True)
        hidden, weight, target = xent_inputs(rows, d, vocab, dtype)
        target[0] = vocab - 1
        hidden.requires_grad_()
        weight.requires_grad_()
        loss = mamba3_amd.linear_cross_entropy(hidden, weight, target, reduction=reduction)
        grad = randn(rows, dtype=torch.float32, seed=5) if reduction == "none" else torch.tensor(1.5, device="cuda")
        dh, dw = torch.autograd.grad(loss, [hidden, weight], grad)
        want = xent_expected(hidden, weight, target, reduction, grad, dtype)
        assert loss.dtype == torch.float32 and dh.dtype == dw.dtype == dtype
        for name, got, w in zip(("loss", "dhidden", "dweight"), (loss, dh, dw), want):
            hold(name, got, w)
        assert not dh[target == -100].any()


@pytest.mark.parametrize("rows,d,vocab", [(4096, 64, 40000), (4096, 768, 8192), (8192, 256, 1000)])
def test_xent_large_tiles_and_pieces(rows, d, vocab):
    """The 256 x 256 tiles; at (4096, 40000) the backward works through two pieces of the vocabulary."""
    print(rows, d, vocab, flush=True)
    hidden, weight, target = xent_inputs(rows, d, vocab, torch.bfloat16)
    hidden.requires_grad_()
    weight.requires_grad_()
    loss = mamba3_amd.linear_cross_entropy(hidden, weight, target)
    got = [loss, *torch.autograd.grad(loss, [hidden, weight])]
    want = xent_expected(hidden, weight, target, "mean", 1.0, torch.bfloat16)
    for name, g, w in zip(("loss", "dhidden", "dweight"), got, want):
        hold(name, g, w)


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp32"])
def test_xent_ignored_rows_may_hold_anything(dtype):
    hidden, weight, target = xent_inputs(50, 40, 90, dtype)
    target[3], target[8], target[20] = -100, -100, -100
    clean = hidden.clone()
    hidden[3], hidden[8], hidden[20, 1] = math.nan, math.inf, -math.inf

    def run(h, reduction):
        h = h.detach().requires_grad_()
        w = weight.detach().requires_grad_()
        loss = mamba3_amd.linear_cross_entropy(h, w, target, reduction=reduction)
        return [loss, *torch.autograd.grad(loss.sum(), [h, w])]

    for reduction in ("mean", "sum", "none"):
        for a, b in zip(run(clean, reduction), run(hidden, reduction)):
            assert torch.isfinite(b).all() and torch.equal(a, b)


def test_xent_no_row_counts():
    hidden, weight, _ = xent_inputs(6, 16, 20, torch.float32)
    target = torch.full((6,), 7, device="cuda")
    hidden.requires_grad_()
    weight.requires_grad_()
    for reduction, want in (("mean", math.nan), ("sum", 0.0)):
        loss = mamba3_amd.linear_cross_entropy(hidden, weight, target, ignore_index=7, reduction=reduction)
        dh, dw = torch.autograd.grad(loss, [hidden, weight])
        assert loss.item() == want or (math.isnan(want) and math.isnan(loss.item()))
        assert not dh.any() and not dw.any()


def test_xent_target_outside_the_vocabulary_is_nan():
    hidden, weight, target = xent_inputs(6, 16, 20, torch.float32, ignored=0.0)
    for bad in (20, -1, 1 << 40, -(1 << 40)):
        target[2] = bad
        h, w = hidden.detach().requires_grad_(), weight.detach().requires_grad_()
        loss = mamba3_amd.linear_cross_entropy(h, w, target, reduction="none")
        assert torch.isnan(loss).tolist() == [i == 2 for i in range(6)]
        dh, dw = torch.autograd.grad(loss.sum(), [h, w])
        assert torch.isnan(dh[2]).all() and torch.isfinite(dh[[0, 1, 3, 4, 5]]).all() and torch.isnan(dw).any()


def test_xent_extreme_logits():
    """Logits of +-1e4 and columns at the type's lowest value: finite, as in 64 bits."""
    for dtype in DTYPES:
        hidden = torch.tensor([[1.0, 0.0], [0.0, 1.0], [1.0, 1.0]], device="cuda", dtype=dtype).requires_grad_()
        low = torch.finfo(dtype).min / 4
        weight = torch.tensor([[1e4, -1e4], [-1e4, 1e4], [low, low], [0.0, 0.0]], device="cuda", dtype=dtype).requires_grad_()
        target = torch.tensor([0, 3, 1], device="cuda")
        loss = mamba3_amd.linear_cross_entropy(hidden, weight, target, reduction="none")
        dh, dw = torch.autograd.grad(loss.sum(), [hidden, weight])
        want = torch.nn.functional.cross_entropy(hidden.double() @ weight.double().t(), target, reduction="none")
        assert torch.allclose(loss.double(), want, rtol=2.0 ** -22, atol=1e-6)
        assert torch.isfinite(dh).all() and torch.isfinite(dw).all()


def test_xent_gradients_wanted_alone_and_batch_dimensions():
    hidden, weight, target = xent_inputs(24, 48, 70, torch.bfloat16)
    want = xent_expected(hidden, weight, target, "mean", 1.0, torch.bfloat16)
    for i, trained in enumerate(((True, False), (False, True))):
        h = hidden.detach().view(2, 3, 4, 48).requires_grad_(trained[0])
        w = weight.detach().clone().requires_grad_(trained[1])
        mamba3_amd.linear_cross_entropy(h, w, target.view(2, 3, 4)).backward()
        got = (h, w)[i].grad
        assert (w, h)[i].grad is None
        hold("gradient", got.reshape(-1, 48), want[1 + i])


def test_xent_strides_and_alignment():
    hidden, weight, target = xent_inputs(33, 40, 51, torch.bfloat16)

    def run(h, w, t):
        h, w = h.detach().requires_grad_(), w.detach().requires_grad_()
        loss = mamba3_amd.linear_cross_entropy(h, w, t)
        return [loss, *torch.autograd.grad(loss, [h, w])]

    off = torch.zeros(hidden.numel() + 3, device="cuda", dtype=hidden.dtype)
    off[3:] = hidden.reshape(-1)
    wide = torch.zeros(33, 2, device="cuda", dtype=torch.long)
    wide[:, 1] = target
    for a, b in zip(run(hidden, weight, target), run(off[3:].view(33, 40), weight.t().contiguous().t(), wide[:, 1])):
        assert torch.equal(a, b)


def test_xent_no_rows():
    weight = torch.ones(5, 8, device="cuda", requires_grad=True)
    hidden = torch.empty(0, 8, device="cuda", requires_grad=True)
    target = torch.empty(0, device="cuda", dtype=torch.long)
    assert math.isnan(mamba3_amd.linear_cross_entropy(hidden, weight, target).item())
    assert mamba3_amd.linear_cross_entropy(hidden, weight, target, reduction="none").shape == (0,)
    mamba3_amd.linear_cross_entropy(hidden, weight, target, reduction="sum").backward()
    assert not weight.grad.any() and hidden.grad.shape == (0, 8)


def test_xent_gradient_against_differences():
    hidden, weight, target = xent_inputs(7, 20, 31, torch.float32)
    target[0] = 4
    h, w = hidden.requires_grad_(), weight.requires_grad_()
    grads = torch.autograd.grad(mamba3_amd.linear_cross_entropy(h, w, target), [h, w])
    want = xent_expected(h, w, target, "mean", 1.0, torch.float32)
    live = target != -100

    def f(a, b):
        z = a @ b.t()
        return (torch.logsumexp(z, 1) - z.gather(1, torch.where(live, target, 0)[:, None])[:, 0])[live].mean().item()

    a, b = h.detach().double(), w.detach().double()
    for i, base in enumerate((a, b)):
        way = randn(*base.shape, dtype=torch.float32, seed=11).double()
        step = 1e-5 * way
        slope = (f(a + step, b) - f(a - step, b) if i == 0 else f(a, b + step) - f(a, b - step)) / 2e-5
        allowed = (want[1 + i].e * way.abs()).sum().item() + 1e-8 * (1 + abs(slope))
        assert abs((grads[i].double() * way).sum().item() - slope) <= allowed


@pytest.mark.parametrize("rows,d,vocab,parts", [(1, 64, 128000, 64), (16, 200, 50021, 48), (16, 64, 128000, 64)])
def test_xent_few_rows_sum_the_vocabulary_in_parts(rows, d, vocab, parts):
    """dhidden of few rows is a sum over the whole vocabulary. All its terms but the last are alike and positive
    (hidden is zero, a column of the weight is one number), so that roundings of one chain of additions fall to the
    same side; cut into parts, a part's chain is vocab / parts long and the parts' sums come to it."""
    print(rows, d, vocab, flush=True)
    weight = (1.0 + torch.rand(1, d, generator=torch.Generator().manual_seed(0)).cuda()).expand(vocab, d).contiguous().requires_grad_()
    hidden = torch.zeros(rows, d, device="cuda", requires_grad=True)
    target = torch.full((rows,), vocab - 1, device="cuda")
    loss = mamba3_amd.linear_cross_entropy(hidden, weight, target, reduction="sum")
    dh, dw = torch.autograd.grad(loss, [hidden, weight])
    lse = math.log(vocab)
    w = weight[0].detach().double()
    # p = 1 / vocab off by lse's own error (its sum: 64 terms in a lane, 500 tiles' pairs) and the exponential's
    e_p = (lse + 4) * 2.0 ** -22 + (64 + vocab / 256 + 2 * lse) * STEP
    # the terms' magnitudes are 2 w in all; the true sum is 0
    bound = 2 * w * (e_p + (vocab / parts + parts + 2) * STEP)
    assert abs(loss.item() - rows * lse) <= rows * lse * e_p
    assert (dh.double().abs() <= bound).all(), (dh.double().abs() / bound).max().item()
    assert not dw.any()  # products with hidden


# ---------------------------------------------------------------- clipping
def _params(shapes, seed=0, std=1.0):
    out = []
    for i, (shape, dtype) in enumerate(shapes):
        p = torch.nn.Parameter(torch.empty(shape, device="cuda", dtype=dtype))
        p.grad = randn(*shape, dtype=dtype, seed=seed + i, std=std)
        out.append(p)
    return out


def check_clip(params, max_norm, kind=2.0):
    before = [p.grad.detach().clone() for p in params]
    each = torch.stack([b.double().abs().max() if kind == math.inf else b.double().square().sum() for b in before if b.numel()])
    norm = (each.max() if kind == math.inf else each.sum().sqrt()).item()
    got = mamba3_amd.clip_grad_norm_(params, max_norm, norm_type=kind)
    assert got.dtype == torch.float32 and got.shape == ()
    assert abs(got.item() - norm) <= STEP * norm
    factor = min(1.0, max_norm / (norm + 1e-6))
    for p, b in zip(params, before):
        if factor == 1.0:
            assert torch.equal(p.grad, b)
        else:
            want = b.double() * factor
            assert ((p.grad.double() - want).abs() <= want.abs() * (HALF[b.dtype] + 2 * STEP) + 1e-38).all()


SHAPES = [(1,), (3,), (8,), (5, 7), (1000,), (32769,), (65536 + 5,), (0,), (300, 513)]


@pytest.mark.parametrize("kind", [2.0, math.inf])
@pytest.mark.parametrize("dtypes", [(torch.float32,), (torch.bfloat16,), (torch.float32, torch.bfloat16)],
                         ids=["fp32", "bf16", "mixed"])
def test_clip(dtypes, kind):
    shapes = [(s, dtypes[i % len(dtypes)]) for i, s in enumerate(SHAPES)]
    for max_norm in (0.5, 1e4, 0.0, math.inf):
        check_clip(_params(shapes), max_norm, kind)


def test_clip_many_tensors_and_one():
    check_clip(_params([((1 + i % 5, 3), DTYPES[i % 3 == 0]) for i in range(700)]), 1.0)
    check_clip(_params([((3 << 20,), torch.float32)]), 1.0)
    (p,) = _params([((17,), torch.float32)])
    check_clip([p], 0.1)
    assert mamba3_amd.clip_grad_norm_(p, 100.0).item() < 0.11  # a single tensor, clipped before


def test_clip_misaligned_strided_and_repeated():
    flat = randn(5000, dtype=torch.bfloat16, seed=1)
    params = []
    at = 1
    for n in (7, 64, 1001, 13):
        p = torch.nn.Parameter(torch.empty(n, device="cuda", dtype=torch.bfloat16))
        p.grad = flat[at:at + n]
        params.append(p)
        at += n
    rest = flat[at:].clone()
    q = torch.nn.Parameter(torch.empty(6, 50, device="cuda"))
    q.grad = randn(50, 6, dtype=torch.float32, seed=2).t()
    params.append(q)
    check_clip(params, 0.25)
    assert torch.equal(flat[at:], rest) and not q.grad.is_contiguous()
    # listed twice: counted and scaled once
    (a,) = _params([((100,), torch.float32)])
    (b,) = _params([((100,), torch.float32)])
    assert torch.equal(mamba3_amd.clip_grad_norm_([a, a], 1.0), mamba3_amd.clip_grad_norm_([b], 1.0))
    assert torch.equal(a.grad, b.grad)


def test_clip_range():
    """Elements whose squares leave fp32's range on either side."""
    for std in (1e30, 1e-30):
        params = _params([((1000,), torch.float32), ((77,), torch.bfloat16)], std=std)
        norm = torch.cat([p.grad.double() for p in params]).norm().item()
        got = mamba3_amd.clip_grad_norm_(params, math.inf).item()
        assert abs(got - norm) <= STEP * norm


def test_clip_nonfinite():
    for value, kind in ((math.nan, 2.0), (math.nan, math.inf), (math.inf, 2.0), (-math.inf, math.inf)):
        params = _params([((100,), torch.float32), ((40000,), torch.float32)])
        params[1].grad[31234] = value
        before = [p.grad.clone() for p in params]
        with pytest.raises(RuntimeError, match="not clipped"):
            mamba3_amd.clip_grad_norm_(params, 1.0, norm_type=kind, error_if_nonfinite=True)
        assert all(torch.equal(p.grad, b) or value != value for p, b in zip(params, before))
        assert torch.equal(params[0].grad, before[0])
        got = mamba3_amd.clip_grad_norm_(params, 1.0, norm_type=kind).item()
        assert math.isnan(got) if math.isnan(value) else got == math.inf
        assert torch.isnan(params[0].grad).all() if math.isnan(value) else not params[0].grad.any()


def test_clip_refuses_shared_memory_and_marks_what_it_writes():
    base = randn(100, dtype=torch.float32, seed=3)
    a, b = torch.nn.Parameter(torch.empty(60, device="cuda")), torch.nn.Parameter(torch.empty(60, device="cuda"))
    a.grad, b.grad = base[:60], base[40:]
    kept = base.clone()
    with pytest.raises(ValueError, match="overlap"):
        mamba3_amd.clip_grad_norm_([a, b], 1.0)
    a.grad = torch.ones(1, device="cuda").expand(60)
    with pytest.raises(ValueError, match="expanded"):
        mamba3_amd.clip_grad_norm_([a], 1.0)
    assert torch.equal(base, kept)
    (p,) = _params([((10,), torch.float32)])
    version = p.grad._version
    mamba3_amd.clip_grad_norm_([p], 0.1)
    assert p.grad._version > version


# ---------------------------------------------------------------- streams, graphs, compilation
def _step(x, weights, head, target):
    """One pass of all three: MLP with its residual, loss, gradients, clipping."""
    y = mamba3_amd.swiglu_mlp(x, *weights, residual=x, scale=0.5)
    loss = mamba3_amd.linear_cross_entropy(y, head, target)
    leaves = [*weights, head]
    for p, g in zip(leaves, torch.autograd.grad(loss, leaves)):
        p.grad.copy_(g)
    norm = mamba3_amd.clip_grad_norm_(leaves, 0.05)
    return loss.detach(), norm


def _step_inputs(seed=0, rows=300):
    t = mlp_inputs(rows, 128, 320, torch.bfloat16, seed=seed)
    x = t["x"]
    weights = [torch.nn.Parameter(t[k]) for k in ("w_gate", "w_up", "w_down")]
    _, head, target = xent_inputs(rows, 128, 1000, torch.bfloat16, seed=seed)
    head = torch.nn.Parameter(head)
    for p in (*weights, head):
        p.grad = torch.zeros_like(p)
    return x, weights, head, target


def test_results_do_not_change_from_run_to_run():
    runs = []
    for _ in range(3):
        x, weights, head, target = _step_inputs(rows=1500)
        runs.append([*_step(x, weights, head, target), *[p.grad for p in (*weights, head)]])
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_on_another_stream():
    want = _step_inputs()
    base = _step(*want)
    got = _step_inputs()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = _step(*got)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(base, out))
    assert all(torch.equal(a.grad, b.grad) for a, b in zip((*want[1], want[2]), (*got[1], got[2])))


def test_captured_step_replays():
    """Two captured training steps (forward, backward, clipping), replayed in turn with eager work
    between, against the eager results for the same inputs."""
    sets = [_step_inputs(seed=s) for s in (0, 100)]
    eager = {}
    for i in range(2):
        for s in (200, 300):
            x, weights, head, target = _step_inputs(seed=100 * i)
            x.copy_(_step_inputs(seed=s)[0])
            eager[i, s] = [t.clone() for t in (*_step(x, weights, head, target), *[p.grad for p in (*weights, head)])]
    graphs = []
    for x, weights, head, target in sets:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _step(x, weights, head, target)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _step(x, weights, head, target)
        graphs.append((graph, out))
    for s in (200, 300, 200):
        for i, (graph, out) in enumerate(graphs):
            x, weights, head, target = sets[i]
            x.copy_(_step_inputs(seed=s)[0])
            graph.replay()
            torch.cuda.synchronize()
            got = [*out, *[p.grad for p in (*weights, head)]]
            assert all(torch.equal(a, b) for a, b in zip(got, eager[i, s]))
            _step(*_step_inputs(seed=7))  # eager work of its own between the replays


# ---------------------------------------------------------------- offsets past 32 bits
def test_mlp_offsets_past_32_bits():
    """h, and what is kept for the backward, pass 4 GiB: the last rows against the definition. Only
    they have a dy, so the weights' gradients are theirs."""
    rows, d, ff, last = (1 << 21) + 37, 64, 1088, 300
    print(rows, d, ff, flush=True)
    t = mlp_inputs(rows, d, ff, torch.bfloat16)
    dy = torch.zeros(rows, d, device="cuda", dtype=torch.bfloat16)
    dy[-last:] = randn(last, d, dtype=torch.bfloat16, seed=9)
    leaves = {k: v.requires_grad_() for k, v in t.items()}
    y = mamba3_amd.swiglu_mlp(**t, scale=0.5)
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))
    end = {k: v.detach()[-last:] if k in ("x", "residual") else v.detach() for k, v in t.items()}
    want = mlp_expected(end, 0.5, dy[-last:], torch.bfloat16)
    hold("y", y[-last:], want["y"])
    for k in leaves:
        hold(k, grads[k][-last:] if k in ("x", "residual") else grads[k], want[k])
    assert not grads["x"][:-last].any()


def test_xent_row_offsets_past_32_bits():
    rows, d, vocab, last = (1 << 25) + 5, 64, 200, 300
    print(rows, d, vocab, flush=True)
    hidden, weight, target = xent_inputs(rows, d, vocab, torch.bfloat16)
    grad = torch.zeros(rows, device="cuda")
    grad[-last:] = randn(last, dtype=torch.float32, seed=5)
    hidden.requires_grad_()
    weight.requires_grad_()
    loss = mamba3_amd.linear_cross_entropy(hidden, weight, target, reduction="none")
    dh, dw = torch.autograd.grad(loss, [hidden, weight], grad)
    want = xent_expected(hidden.detach()[-last:], weight, target[-last:], "none", grad[-last:], torch.bfloat16)
    for name, got, w in zip(("loss", "dhidden", "dweight"), (loss[-last:], dh[-last:], dw), want):
        hold(name, got, w)
    assert not dh[:-last].any()


def test_xent_vocabulary_offsets_past_32_bits():
    """A weight of 4 GiB whose last rows are not zero, and hold the targets."""
    rows, d, vocab, last = 5, 64, (1 << 25) + 3, 70
    print(rows, d, vocab, flush=True)
    hidden, end, target = xent_inputs(rows, d, last, torch.bfloat16, ignored=0.0)
    weight = torch.zeros(vocab, d, device="cuda", dtype=torch.bfloat16)
    weight[-last:] = end * 4  # exact; some logits of these rows outweigh the zeros of all others
    hidden.requires_grad_()
    weight.requires_grad_()
    loss = mamba3_amd.linear_cross_entropy(hidden, weight, target + vocab - last, reduction="sum")
    dh, dw = torch.autograd.grad(loss, [hidden, weight])
    h, w = Num(hidden), Num(weight.detach()[-last:])
    z = h.dot(w)
    lse = torch.logaddexp(torch.logsumexp(z.v, 1), torch.full((rows,), math.log(vocab - last), device="cuda").double())[:, None]
    # a row's sum: at most 256 terms in a lane's and a tile's order, then the tiles' pairs one by one
    e_lse = z.e.amax(1, keepdim=True) + (64 + vocab / 64 + (z.top.amax(1, keepdim=True) + 4) * 2) * STEP + lse.abs() * STEP * 2
    at = target[:, None]
    want = (lse - z.v.gather(1, at)).sum()
    assert abs(loss.item() - want.item()) <= (e_lse + z.e.gather(1, at) + 2 * STEP * (lse.abs() + z.top.gather(1, at))).sum().item()
    p = torch.exp(z.v - lse)
    dz = Num(p - torch.zeros_like(p).scatter_(1, at, 1.0), p * torch.expm1(z.e + e_lse + ((z.v - lse).abs() + 4) * 2.0 ** -22) + STEP)
    dz = dz.rounded(torch.bfloat16)
    # the other rows of the weight are zero: they add nothing to dhidden
    hold("dhidden", dh, dz.dot(w.t()).rounded(torch.bfloat16))
    hold("dweight", dw[-last:], dz.t().dot(h.t()).rounded(torch.bfloat16))
    rest = torch.exp(-lse) * torch.ones(1, 1000, device="cuda").double()
    rest = Num(rest, rest * torch.expm1(e_lse + (lse.abs() + 4) * 2.0 ** -22)).rounded(torch.bfloat16)
    for begin in (0, (1 << 25) - 2000):
        hold("dweight", dw[begin:begin + 1000], rest.t().dot(h.t()).rounded(torch.bfloat16))


def test_clip_offsets_past_32_bits():
    n = (1 << 32) + 12345
    print(n, flush=True)
    p = torch.nn.Parameter(torch.empty(n, device="cuda", dtype=torch.bfloat16))
    p.grad = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    p.grad[0], p.grad[1 << 32], p.grad[-1] = 2.0, 3.0, 6.0
    assert mamba3_amd.clip_grad_norm_(p, 3.5).item() == 7.0
    # the factor is 0.5 but for 1e-6 / 7: the halves are the nearest bf16
    assert (p.grad[0].item(), p.grad[1 << 32].item(), p.grad[-1].item()) == (1.0, 1.5, 3.0)
    assert p.grad.count_nonzero().item() == 3


def test_compiled_for_other_row_counts():
    x, weights, head, target = _step_inputs()

    def f(x, target):
        return mamba3_amd.linear_cross_entropy(mamba3_amd.swiglu_mlp(x, *weights, residual=x), head, target)

    leaves = [*weights, head]
    step = torch.compile(f, fullgraph=True, dynamic=True)
    for n in (x.shape[0], x.shape[0] // 2 + 1, 3):
        want = torch.autograd.grad(f(x[:n], target[:n]), leaves)
        got = torch.autograd.grad(step(x[:n], target[:n]), leaves)
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_compiled_step():
    x, weights, head, target = _step_inputs()

    def f(x, target):
        y = mamba3_amd.swiglu_mlp(x, *weights, residual=x, scale=0.5)
        return mamba3_amd.linear_cross_entropy(y, head, target)

    leaves = [*weights, head]
    want = torch.autograd.grad(f(x, target), leaves)
    got = torch.autograd.grad(torch.compile(f, fullgraph=True)(x, target), leaves)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_autocast():
    """fp32 tensors under bf16 autocast: the products of their bf16 copies, the residual added in fp32."""
    t = mlp_inputs(20, 64, 96, torch.float32)
    low = {k: v.bfloat16() for k, v in t.items()}
    hidden, weight, target = xent_inputs(20, 64, 50, torch.float32)
    args = [low[k] for k in ("x", "w_gate", "w_up", "w_down")]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = mamba3_amd.swiglu_mlp(**t, scale=0.5)
        loss = mamba3_amd.linear_cross_entropy(hidden, weight, target)
    assert y.dtype == torch.float32
    assert torch.equal(y, t["residual"] + mamba3_amd.swiglu_mlp(*args, scale=0.5))
    assert torch.equal(loss, mamba3_amd.linear_cross_entropy(hidden.bfloat16(), weight.bfloat16(), target))
    lm = _lm(torch.float32).fuse_mlp()
    ids = torch.randint(300, (2, 20), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = lm.loss(ids, ids)
    loss.backward()
    assert loss.dtype == torch.float32 and torch.isfinite(loss) and lm.embedding.weight.grad.dtype == torch.float32


def test_two_streams_at_once():
    """The same two steps side by side on two streams, and after one another: nothing is shared."""
    sets = [_step_inputs(seed=s, rows=900) for s in (0, 100)]
    want = [[t.clone() for t in (*_step(*_step_inputs(seed=s, rows=900)),)] for s in (0, 100)]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = []
    for st, args in zip(streams, sets):
        with torch.cuda.stream(st):
            got.append(_step(*args))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_second_backward_and_changed_inputs_are_refused():
    t = mlp_inputs(6, 16, 24, torch.float32)
    x = t["x"].requires_grad_()
    y = mamba3_amd.swiglu_mlp(**t)
    (g,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    hidden, weight, target = xent_inputs(6, 16, 20, torch.float32)
    loss = mamba3_amd.linear_cross_entropy(hidden, weight.requires_grad_(), target)
    with torch.no_grad():
        weight.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


# ---------------------------------------------------------------- the language model
def _lm(dtype, **kw):
    torch.manual_seed(0)
    return mamba3_amd.KulaMambaLM(300, 128, n_layers=2, d_state=32, headdim=32, **kw).cuda().to(dtype)


@pytest.mark.parametrize("checkpointing", [False, True])
def test_lm_loss_equals_forward(checkpointing):
    """fp32: the same loss and gradients as the path that keeps the logits. Both are fp32 passes over
    the same layers; the new operators' own error is bounded above, the two paths' joint error by the
    1e-4 that the fp32 layer's gradients are held to against 64 bits."""
    ids = torch.randint(300, (3, 50), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    labels = ids.clone()
    labels[1, 20:] = -100
    lm = _lm(torch.float32, gradient_checkpointing=checkpointing).train()
    a = lm(ids, labels)["loss"]
    ga = torch.autograd.grad(a, list(lm.parameters()))
    b = lm.fuse_mlp().loss(ids, labels)
    gb = torch.autograd.grad(b, list(lm.parameters()))
    assert abs(a.item() - b.item()) <= 1e-5 * abs(a.item())
    for (name, _), x, y in zip(lm.named_parameters(), ga, gb):
        assert (x - y).norm() <= 1e-4 * x.norm(), name


def test_lm_training_steps_in_bf16():
    lm = _lm(torch.bfloat16).train().fuse_mlp()
    opt = torch.optim.SGD(lm.parameters(), lr=0.1)
    ids = torch.randint(300, (2, 40), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    for _ in range(3):
        opt.zero_grad()
        loss = lm.loss(ids, ids)
        loss.backward()
        norm = mamba3_amd.clip_grad_norm_(lm.parameters(), 1.0)
        opt.step()
        assert math.isfinite(loss.item()) and math.isfinite(norm.item())
    with pytest.raises(ValueError, match="labels"):
        lm.loss(ids, ids[:, :-1])


def test_lm_fused_serving_and_switching_back():
    """prefill, step and generate with the fused MLP, and bitwise what was there once it is off."""
    lm = _lm(torch.bfloat16).eval()
    ids = torch.randint(300, (12, 33), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    with torch.no_grad():
        before = lm(ids)["logits"]
        fused = lm.fuse_mlp()(ids)["logits"]
        tokens = lm.generate(ids, max_new_tokens=4, temperature=0)
        after = lm.fuse_mlp(False)(ids)["logits"]
    assert torch.equal(before, after) and tokens.shape == (12, 37)
    # bf16 activations of two layers: a few roundings of 2^-8 each
    assert (fused.float() - before.float()).norm() <= 8 * 2.0 ** -8 * before.float().norm()
