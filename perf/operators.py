"""Cases of the training operators: the gated MLP with its residual, the vocabulary projection with its
softmax cross entropy, and the clipping of gradients by their global norm.

`run` computes a case either in elementary torch operations (`own` false) or with this package's kernels
(`own` true); `exact` computes it in 64 bits. Sizes are those of this repository's language model: d_model
768 and 2048 with the hidden width that KulaMambaBlock derives from them, 32000 tokens, 24 layers.
"""

import math

import torch
import torch.nn.functional as F

own = False

_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _width(d):
    """The MLP's hidden width that KulaMambaBlock takes at its default expansion."""
    return int(d * 2.667 / 64 + 1) * 64


def listed():
    return [
        # a serving batch of 24 single tokens (or one short prompt) through one layer's MLP, no gradients
        {"name": "mlp_fwd_d768_M24", "op": "mlp", "dtype": "bf16", "rows": 24, "d": 768, "ff": 2112, "train": False},
        # one layer's MLP in a training step of 4 sequences of 2048 tokens
        {"name": "mlp_train_d768_M8192", "op": "mlp", "dtype": "bf16", "rows": 8192, "d": 768, "ff": 2112, "train": True},
        # the same at the larger layer
        {"name": "mlp_train_d2048_M8192", "op": "mlp", "dtype": "bf16", "rows": 8192, "d": 2048, "ff": 5504, "train": True},
        # fp32 parameters, as a module has them by default; a ragged number of tokens
        {"name": "mlp_train_fp32_d768_M1000", "op": "mlp", "dtype": "fp32", "rows": 1000, "d": 768, "ff": 2112, "train": True},
        # widths that no tile or 16-byte piece divides
        {"name": "mlp_train_odd_d500_M777", "op": "mlp", "dtype": "bf16", "rows": 777, "d": 500, "ff": 1363, "train": True},
        # the language model's loss in a training step of 4 sequences of 2048 tokens
        {"name": "ce_train_d768_V32000_M8192", "op": "ce", "dtype": "bf16", "rows": 8192, "d": 768, "vocab": 32000, "train": True, "reduction": "mean"},
        # a large vocabulary at the larger layer: the largest case
        {"name": "ce_train_d2048_V128000_M4096", "op": "ce", "dtype": "bf16", "rows": 4096, "d": 2048, "vocab": 128000, "train": True, "reduction": "mean"},
        # a byte vocabulary and the tests' tiny model in fp32: a small call
        {"name": "ce_train_fp32_d64_V256_M1024", "op": "ce", "dtype": "fp32", "rows": 1024, "d": 64, "vocab": 256, "train": True, "reduction": "mean"},
        # scoring of one text: each token's loss, no gradients, an odd vocabulary
        {"name": "ce_score_d768_V50021_M1000", "op": "ce", "dtype": "bf16", "rows": 1000, "d": 768, "vocab": 50021, "train": False, "reduction": "none"},
        # all gradients of the 24-layer model, fp32
        {"name": "clip_fp32_d768_L24", "op": "clip", "dtype": "fp32", "d": 768, "layers": 24, "vocab": 32000},
        # the same model in bf16 with half the layers
        {"name": "clip_bf16_d768_L12", "op": "clip", "dtype": "bf16", "d": 768, "layers": 12, "vocab": 32000},
        # the tests' tiny model: a few small tensors
        {"name": "clip_fp32_d64_L2", "op": "clip", "dtype": "fp32", "d": 64, "layers": 2, "vocab": 256},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["mlp", "mlp", "ce", "ce", "clip"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    d = rng.choice([64, 128, 256, 512, 768, 1024, 1536, 2048, rng.randint(40, 2048)])
    if op == "clip":
        return {"op": op, "dtype": dtype, "d": d, "layers": rng.randint(1, max(1, min(24, 24 * 768 * 768 // (d * d)))), "vocab": _log_int(rng, 200, 32000)}
    train = rng.random() < 0.75
    most = 1 << 33 if dtype == "fp32" else 1 << 36 if op == "mlp" else 1 << 39  # rows * d * width of the dearest draw
    if op == "mlp":
        ff = _width(d) if rng.random() < 0.7 else rng.randint(max(8, d), 3 * d)
        rows = _log_int(rng, 1, max(1, min(16384, most // (d * ff))))
        return {"op": op, "dtype": dtype, "rows": rows, "d": d, "ff": ff, "train": train}
    vocab = _log_int(rng, 200, 128000)
    rows = _log_int(rng, 1, max(1, min(16384, most // (d * vocab))))
    return {"op": op, "dtype": dtype, "rows": rows, "d": d, "vocab": vocab, "train": train,
            "reduction": rng.choice(["mean", "sum"]) if train else rng.choice(["mean", "none"])}


def _shapes(case):
    """Shapes of the gradients of a KulaMambaLM of these sizes (d_state 128, headdim 64, rank 2), its embedding last."""
    d = case["d"]
    inner, state, rank = 2 * d, 128, 2
    heads = max(1, inner // 64)
    ff = _width(d)
    wide = 2 * inner + 2 * state * rank + 2 * heads + state // 2
    small = [(heads,)] * 3 + [(state * rank,)] * 2 + [(1, state, rank)] * 2 + [(heads, 64, rank)] * 3
    layer = [(d,), *small, (wide, d), (d, inner), (d,), (ff, d), (ff, d), (d, ff)]
    return layer * case["layers"] + [(d,), (case["vocab"], d)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = _TYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * std).to(dt)

    if case["op"] == "clip":
        # gradients lie in one flat buffer, as they do for bucketed data parallelism, each on a 512-byte border
        shapes = _shapes(case)
        pad = 512 // dt.itemsize
        sizes = [math.prod(s) for s in shapes]
        starts = [0]
        for n in sizes:
            starts.append(starts[-1] + -(-n // pad) * pad)
        flat = normal(starts[-1], std=0.01)
        params = []
        for s, n, at in zip(shapes, sizes, starts):
            flat[at + n:at + -(-n // pad) * pad] = 0
            p = torch.nn.Parameter(torch.empty(s, device="cuda", dtype=dt))
            p.grad = flat[at:at + n].view(s)
            params.append(p)
        return {"op": "clip", "flat": flat, "params": params, "max_norm": 1.0}
    rows, d = case["rows"], case["d"]
    if case["op"] == "mlp":
        ff, train = case["ff"], case["train"]
        st = {"op": "mlp", "train": train, "scale": 1 / math.sqrt(48),
              "x": normal(rows, d), "w_gate": normal(ff, d, std=0.02), "w_up": normal(ff, d, std=0.02),
              "w_down": normal(d, ff, std=0.02), "residual": normal(rows, d)}
        if train:
            st["dy"] = normal(rows, d, std=1e-2)
            for k in ("x", "w_gate", "w_up", "w_down"):
                st[k].requires_grad_()
        return st
    vocab, train = case["vocab"], case["train"]
    weight = normal(vocab, d, std=0.02)
    target = torch.randint(vocab, (rows,), generator=gen, device="cuda")
    # hidden states lean to their token by different amounts, from an untrained model's to a sure one's
    lean = torch.rand(rows, 1, generator=gen, device="cuda") * 20
    pick = weight[target].float()
    hidden = (torch.randn(rows, d, generator=gen, device="cuda") + lean * pick / pick.norm(dim=1, keepdim=True)).to(dt)
    # padding: a tenth of the tokens does not count (the first one always does)
    skip = torch.rand(rows, generator=gen, device="cuda") < 0.1
    skip[0] = False
    target = torch.where(skip, -100, target)
    if train:
        hidden.requires_grad_()
        weight.requires_grad_()
    return {"op": "ce", "train": train, "reduction": case["reduction"], "hidden": hidden, "weight": weight, "target": target}


def _plain_mlp(st):
    dt = st["x"].dtype
    x, wg, wu, wd = (st[k].detach().float() for k in ("x", "w_gate", "w_up", "w_down"))
    g, u = x @ wg.t(), x @ wu.t()
    s = 1 / (1 + torch.exp(-g))
    h = g * s * u
    y = (st["residual"].float() + st["scale"] * (h @ wd.t())).to(dt)
    if not st["train"]:
        return {"y": y}
    dy = st["dy"].float() * st["scale"]
    dh = dy @ wd
    du = dh * g * s
    dg = dh * u * s * (1 + g * (1 - s))
    return {"y": y, "dx": (dg @ wg + du @ wu).to(dt), "dw_gate": (dg.t() @ x).to(dt), "dw_up": (du.t() @ x).to(dt), "dw_down": (dy.t() @ h).to(dt)}


def _plain_ce(st):
    dt = st["hidden"].dtype
    hidden, weight, target = st["hidden"].detach().float(), st["weight"].detach().float(), st["target"]
    valid = target != -100
    at = torch.where(valid, target, 0)[:, None]
    logits = hidden @ weight.t()
    top = logits.amax(1, keepdim=True)
    lse = top + torch.exp(logits - top).sum(1, keepdim=True).log()
    loss = torch.where(valid, (lse - logits.gather(1, at))[:, 0], 0)
    share = valid.float()
    if st["reduction"] == "mean":
        share = share / valid.sum()
        loss = loss.sum(dtype=torch.float64).float() / valid.sum()
    elif st["reduction"] == "sum":
        loss = loss.sum(dtype=torch.float64).float()
    if not st["train"]:
        return {"loss": loss}
    dl = logits.sub_(lse).exp_()
    dl.scatter_add_(1, at, torch.full_like(lse, -1.0))
    dl.mul_(share[:, None])
    return {"loss": loss, "dhidden": (dl @ weight).to(dt), "dweight": (dl.t() @ hidden).to(dt)}


def _plain_clip(st):
    flat = st["flat"]
    norm = flat.float().square().sum(dtype=torch.float64).sqrt()
    flat.copy_(flat.float() * torch.clamp(st["max_norm"] / (norm + 1e-6), max=1.0).float())
    return {"norm": norm.float(), "grads": flat}


def run(state):
    if state["op"] == "clip":
        if own:
            import mamba3_amd
            out = {"norm": mamba3_amd.clip_grad_norm_(state["params"], state["max_norm"]), "grads": state["flat"]}
        else:
            out = _plain_clip(state)
        # the next pass meets what this one left, not the next step's new gradients: under a bound a little lower it still has to scale them
        state["max_norm"] *= 0.9999
        return out
    if not own:
        return _plain_mlp(state) if state["op"] == "mlp" else _plain_ce(state)
    import mamba3_amd
    if state["op"] == "mlp":
        leaves = [state[k] for k in ("x", "w_gate", "w_up", "w_down")]
        with torch.set_grad_enabled(state["train"]):
            y = mamba3_amd.swiglu_mlp(*leaves, residual=state["residual"], scale=state["scale"])
        if not state["train"]:
            return {"y": y}
        dx, dg, du, dd = torch.autograd.grad(y, leaves, state["dy"])
        return {"y": y.detach(), "dx": dx, "dw_gate": dg, "dw_up": du, "dw_down": dd}
    with torch.set_grad_enabled(state["train"]):
        loss = mamba3_amd.linear_cross_entropy(state["hidden"], state["weight"], state["target"], reduction=state["reduction"])
    if not state["train"]:
        return {"loss": loss}
    dh, dw = torch.autograd.grad(loss, [state["hidden"], state["weight"]])
    return {"loss": loss.detach(), "dhidden": dh, "dweight": dw}


def work(case):
    size = _TYPES[case["dtype"]].itemsize
    if case["op"] == "clip":
        n = sum(math.prod(s) for s in _shapes(case))
        return {"bytes": 2 * n * size, "flops": 3 * n}
    m, d = case["rows"], case["d"]
    if case["op"] == "mlp":
        one = 2 * m * d * case["ff"]
        weights = 3 * d * case["ff"]
        if not case["train"]:
            return {"bytes": size * (weights + 3 * m * d), "flops": 3 * one}
        return {"bytes": size * (2 * weights + 5 * m * d), "flops": 9 * one}
    one = 2 * m * d * case["vocab"]
    ins = size * (m * d + case["vocab"] * d) + 8 * m
    if not case["train"]:
        return {"bytes": ins + 4 * m, "flops": one}
    return {"bytes": ins + size * (m * d + case["vocab"] * d), "flops": 3 * one}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "clip":
        norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(p.grad.double()) for p in st["params"]]))
        share = min(1.0, st["max_norm"] / (norm.item() + 1e-6))
        return {"norm": norm, "grads": st["flat"].double() * share}
    if case["op"] == "mlp":
        x, wg, wu, wd = (st[k].detach().double().requires_grad_(st["train"]) for k in ("x", "w_gate", "w_up", "w_down"))
        y = st["residual"].double() + st["scale"] * F.linear(F.silu(F.linear(x, wg)) * F.linear(x, wu), wd)
        if not st["train"]:
            return {"y": y}
        y.backward(st["dy"].double())
        return {"y": y.detach(), "dx": x.grad, "dw_gate": wg.grad, "dw_up": wu.grad, "dw_down": wd.grad}
    hidden, weight = (st[k].detach().double().requires_grad_(st["train"]) for k in ("hidden", "weight"))
    loss = F.cross_entropy(F.linear(hidden, weight), st["target"], ignore_index=-100, reduction=st["reduction"])
    if not st["train"]:
        return {"loss": loss}
    loss.backward()
    return {"loss": loss.detach(), "dhidden": hidden.grad, "dweight": weight.grad}
