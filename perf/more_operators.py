"""Cases of the operators that serve a language model from 4-bit weights: the root-mean-square norm with the
residual's addition (differentiable, or with its output in microscaled 8 bits), microscaled quantisation, the
product with 4-bit weights, and the choice of the next token from given random numbers.

`run` computes a case either in elementary torch operations (`own` false) or with this package's kernels
(`own` true); `exact` computes it in 64 bits. Sizes are those of this repository's language model: d_model
768 and 2048 with the widths that its layers derive from them, 32000 tokens; generic ones beside them.

Microscaled values (blocks of 32 along k share a power of two): `data` has a row of kp elements for each row, kp
being k rounded up to 128, 8 bits each (e4m3) or 4 (e2m1, the even k in a byte's low half); `scales` (rows, kp / 32)
holds each block's exponent plus 127, 255 where the block held an infinity or NaN. The exponent is the smallest under
which the block's largest magnitude rounds to a value of the element type, 0 for a block of zeros.
"""

import math

import torch
import torch.nn.functional as F

own = False

_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
_EPS = 1e-5


def listed():
    return [
        # a decode batch of 64 tokens through one norm of a block, output in 8 bits for the projection behind it
        {"name": "norm_mx_d768_M64", "op": "norm", "dtype": "bf16", "rows": 64, "d": 768, "out": "e4m3", "train": False},
        # the same in the prefill of 8 prompts of 2048 tokens at the larger layer
        {"name": "norm_mx_d2048_M16384", "op": "norm", "dtype": "bf16", "rows": 16384, "d": 2048, "out": "e4m3", "train": False},
        # a block's second norm in a training step of 4 sequences of 2048 tokens, forward and backward
        {"name": "norm_train_d768_M8192", "op": "norm", "dtype": "bf16", "rows": 8192, "d": 768, "out": "same", "train": True},
        # fp32 parameters, a width that no 16-byte piece divides, a ragged number of tokens
        {"name": "norm_train_fp32_d501_M777", "op": "norm", "dtype": "fp32", "rows": 777, "d": 501, "out": "same", "train": True},
        # the vocabulary projection's weight to 4 bits, once per model
        {"name": "quant_e2m1_d768_V32000", "op": "quant", "dtype": "bf16", "rows": 32000, "k": 768, "format": "e2m1", "gated": False},
        # the hidden activations of the gated MLP of 8192 tokens to 8 bits
        {"name": "quant_gated_e4m3_ff2112_M8192", "op": "quant", "dtype": "bf16", "rows": 8192, "k": 2112, "format": "e4m3", "gated": True},
        # in_proj of one decode step of 4 sequences: the activations are quantised within the call
        {"name": "linear_d768_N3696_M4", "op": "linear", "rows": 4, "k": 768, "n": 3696, "x": "bf16", "residual": False, "out": "bf16"},
        # the logits of a decode batch of 16 at a large vocabulary: the weight's read
        {"name": "linear_d2048_V128000_M16", "op": "linear", "rows": 16, "k": 2048, "n": 128000, "x": "e4m3", "residual": False, "out": "bf16"},
        # sizes that no tile or block of 32 divides, with a residual
        {"name": "linear_k500_N1363_M777", "op": "linear", "rows": 777, "k": 500, "n": 1363, "x": "e4m3", "residual": True, "out": "bf16"},
        # gate and up projections of a prefill of 8192 tokens at the larger layer: the largest case
        {"name": "linear_d2048_N11008_M8192", "op": "linear", "rows": 8192, "k": 2048, "n": 11008, "x": "e4m3", "residual": False, "out": "bf16"},
        # the next tokens of 4 sequences
        {"name": "sample_V32000_R4", "op": "sample", "dtype": "bf16", "rows": 4, "vocab": 32000, "temperature": 0.8, "top_k": 50, "top_p": 0.95, "min_p": 0.0, "each": False, "logprob": False},
        # a serving batch at a large vocabulary, each request with settings of its own; the chosen tokens' log probabilities too
        {"name": "sample_V128000_R256", "op": "sample", "dtype": "fp32", "rows": 256, "vocab": 128000, "temperature": 1.0, "top_k": 0, "top_p": 0.9, "min_p": 0.02, "each": True, "logprob": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "quant", "linear", "linear", "linear", "sample", "sample"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    width = lambda lo, hi: rng.choice([_log_int(rng, lo, hi), 64 * max(1, _log_int(rng, lo, hi) // 64)])  # noqa: E731
    if op == "norm":
        d = width(40, 8192)
        rows = _log_int(rng, 1, max(1, min(65536, (1 << 25) // d)))
        out = rng.choice(["same", "same", "e4m3"])
        return {"op": op, "dtype": dtype, "rows": rows, "d": d, "out": out, "train": out == "same" and rng.random() < 0.75}
    if op == "quant":
        k = width(20, 8192)
        return {"op": op, "dtype": dtype, "rows": _log_int(rng, 1, max(1, min(65536, (1 << 25) // k))), "k": k, "format": rng.choice(["e2m1", "e4m3"]), "gated": rng.random() < 0.4}
    if op == "linear":
        k, n = width(40, 8192), width(40, 32000)
        rows = _log_int(rng, 1, max(1, min(16384, (1 << 36) // (k * n))))
        x = rng.choice(["bf16", "e4m3", "e4m3", "e2m1", "fp32"])
        return {"op": op, "rows": rows, "k": k, "n": n, "x": x, "residual": rng.random() < 0.5, "out": "fp32" if x == "fp32" else "bf16"}
    vocab = _log_int(rng, 200, 128000)
    rows = _log_int(rng, 1, max(1, min(512, (1 << 24) // vocab)))
    return {"op": op, "dtype": dtype, "rows": rows, "vocab": vocab, "temperature": rng.choice([1.0, round(rng.uniform(0.3, 1.5), 2)]),
            "top_k": rng.choice([0, 0, 1, _log_int(rng, 2, 2000)]), "top_p": rng.choice([1.0, round(rng.uniform(0.3, 0.99), 2)]),
            "min_p": rng.choice([0.0, 0.0, round(rng.uniform(0.01, 0.3), 2)]), "each": rng.random() < 0.5, "logprob": rng.random() < 0.5}


# ------------------------------------------------------------------ microscaled values, plain
_MOST = {"e2m1": 2, "e4m3": 8}        # exponent of the largest element
_BITS = {"e2m1": 4, "e4m3": 8}


def _blocks(x):
    """fp32 rows, padded to whole 128 columns, in blocks of 32: (rows, kp / 32, 32)."""
    return F.pad(x, (0, -x.shape[-1] % 128)).unflatten(-1, (-1, 32))


def _to_grid(x, fmt):
    """Blocks of fp32 values -> (their element values under the block's scale, exponents, whether the block is finite)."""
    top = x.abs().amax(-1)
    fine = torch.isfinite(top)
    some = torch.where(fine & (top > 0), top, 1.0)
    e = torch.frexp(some).exponent - 1 - _MOST[fmt]
    last = torch.ldexp(some, -e)
    e = e + ((last >= 7) if fmt == "e2m1" else (last > 464)).int()
    e = torch.where(top > 0, e.clamp(min=-127), 0)
    v = torch.ldexp(torch.where(fine[..., None], x, 0.0), -e[..., None])
    low = 0 if fmt == "e2m1" else -6
    step = (torch.frexp(v).exponent - 1).clamp(min=low) - (1 if fmt == "e2m1" else 3)
    return torch.ldexp(torch.round(torch.ldexp(v, -step)), step), e, fine


def _values(x, fmt):
    """The fp32 values that microscaled x stands for, (rows, k)."""
    v, e, fine = _to_grid(_blocks(x), fmt)
    v = torch.where(fine[..., None], torch.ldexp(v, e[..., None]), float("nan"))
    return v.flatten(-2)[..., :x.shape[-1]]


def _stored(x, fmt):
    """Microscaled x as (data, scales)."""
    v, e, fine = _to_grid(_blocks(x), fmt)
    scales = torch.where(fine, e + 127, 255).to(torch.uint8)
    if fmt == "e4m3":
        return v.flatten(-2).to(torch.float8_e4m3fn).view(torch.uint8), scales
    m = v.abs().flatten(-2)
    code = torch.where(m < 2, m * 2, torch.where(m < 4, m + 2, m / 2 + 4)).to(torch.uint8) | (torch.signbit(v.flatten(-2)).to(torch.uint8) << 3)
    return code[..., ::2] | (code[..., 1::2] << 4), scales


def _held(data, scales, fmt, k):
    """The fp32 values of stored ones, (rows, k)."""
    if fmt == "e4m3":
        v = data.view(torch.float8_e4m3fn).float()
    else:
        code = torch.stack((data & 15, data >> 4), -1).flatten(-2).int()
        v = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=data.device)[code]
    e = scales.int() - 127
    v = torch.where((e < 128)[..., None], torch.ldexp(v.unflatten(-1, (-1, 32)), e[..., None]), float("nan"))
    return v.flatten(-2)[..., :k]


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.bfloat16):
        return (torch.randn(*shape, generator=gen, device="cuda") * std).to(dtype)

    op = case["op"]
    st = dict(case)
    if op == "norm":
        dt, rows, d = _TYPES[case["dtype"]], case["rows"], case["d"]
        # a residual stream: a few columns are an order larger than the rest
        wide = 1 + 12 * (torch.rand(d, generator=gen, device="cuda") < 0.01)
        st |= {"x": normal(rows, d, std=0.7, dtype=dt), "residual": (torch.randn(rows, d, generator=gen, device="cuda") * wide).to(dt),
               "weight": (1 + 0.2 * torch.randn(d, generator=gen, device="cuda")).to(dt), "scale": 1 / math.sqrt(48)}
        if case["train"]:
            st |= {"dtotal": normal(rows, d, std=1e-2, dtype=dt), "dy": normal(rows, d, std=1e-2, dtype=dt)}
            for key in ("x", "residual", "weight"):
                st[key].requires_grad_()
    elif op == "quant":
        dt, k = _TYPES[case["dtype"]], case["k"] * (2 if case["gated"] else 1)
        # rows differ in size, as weights' and activations' do
        st["x"] = (torch.randn(case["rows"], k, generator=gen, device="cuda") * torch.exp(torch.randn(case["rows"], 1, generator=gen, device="cuda"))).to(dt)
    elif op == "linear":
        rows, k, n = case["rows"], case["k"], case["n"]
        dt = _TYPES[case["out"]]
        x = torch.randn(rows, k, generator=gen, device="cuda") * torch.exp(0.5 * torch.randn(rows, 1, generator=gen, device="cuda"))
        st["x_in"] = x.to(_TYPES[case["x"]]) if case["x"] in _TYPES else _stored(x, case["x"])
        st["w"] = _stored(normal(n, k, std=0.02, dtype=torch.float32), "e2m1")  # laid out once, as a program keeps it
        st["res"] = normal(rows, n, dtype=dt) if case["residual"] else None
        st["scale"] = 1 / math.sqrt(48) if case["residual"] else 1.0
    else:
        rows, vocab = case["rows"], case["vocab"]
        z = torch.randn(rows, vocab, generator=gen, device="cuda") * 2.5
        # a few likely tokens a row; a tenth of the rows have most of the vocabulary masked away
        likely = torch.randint(vocab, (rows, 8), generator=gen, device="cuda")
        z.scatter_(1, likely, 6 + 6 * torch.rand(rows, 8, generator=gen, device="cuda"))
        masked = (torch.rand(rows, 1, generator=gen, device="cuda") < 0.1) & (torch.rand(rows, vocab, generator=gen, device="cuda") < 0.99)
        masked[:, 0] = False
        st["logits"] = z.masked_fill_(masked, float("-inf")).to(_TYPES[case["dtype"]])
        st["u"] = torch.rand(rows, generator=gen, device="cuda")
        if case["each"]:
            r = lambda: torch.rand(rows, generator=gen, device="cuda")  # noqa: E731
            # one request in sixteen is greedy, one in four does not bound k
            st["temperature"] = torch.where(r() < 1 / 16, 0.0, case["temperature"] * (0.5 + r()))
            st["top_k"] = torch.where(r() < 0.25, 0, (r() * 2 * case["top_k"]).ceil().int())
            st["top_p"] = 1 - (1 - case["top_p"]) * 2 * r()
            st["min_p"] = case["min_p"] * 2 * r()
    return st


# ------------------------------------------------------------------ plain forms
def _plain_norm(st):
    dt, d = st["x"].dtype, st["d"]
    x, res, w = (st[key].detach().float() for key in ("x", "residual", "weight"))
    total = (res + st["scale"] * x).to(dt)
    t = total.float()
    r = 1 / torch.sqrt(t.square().sum(1, keepdim=True) / d + _EPS)
    y = t * r * w
    if st["out"] != "same":
        return {"total": total, "y": _values(y, st["out"]).to(torch.bfloat16)}
    out = {"total": total, "y": y.to(dt)}
    if st["train"]:
        dy = st["dy"].float()
        g = dy * w
        dt_ = st["dtotal"].float() + r * g - t * (r * r * r * (g * t).sum(1, keepdim=True) / d)
        out |= {"dx": (dt_ * st["scale"]).to(dt), "dresidual": dt_.to(dt), "dweight": (dy * t * r).sum(0).to(dt)}
    return out


def _plain_quant(st):
    x = st["x"].float()
    if st["gated"]:
        g, u = x.chunk(2, 1)
        x = g / (1 + torch.exp(-g)) * u
    return {"values": _values(x, st["format"]).to(torch.bfloat16)}


def _plain_linear(st):
    x, w = st["x_in"], _held(*st["w"], "e2m1", st["k"])
    x = _values(x.float(), "e4m3") if torch.is_tensor(x) else _held(*x, st["x"], st["k"])
    y = x @ w.t()
    if st["res"] is not None:
        y = st["res"].float() + st["scale"] * y
    return {"y": y.to(_TYPES[st["out"]])}


def _column(v, like):
    """A setting as a column of 64-bit numbers."""
    return v.double()[:, None] if torch.is_tensor(v) else torch.full_like(like, v)


def _plain_sample(st):
    z, order = torch.sort(st["logits"].double(), dim=1, descending=True, stable=True)
    top = z[:, :1]
    t, k, p, m = (_column(st[key], top) for key in ("temperature", "top_k", "top_p", "min_p"))
    mass = torch.exp((z - top) / torch.where(t > 0, t, 1.0))
    rank = torch.arange(z.shape[1], device=z.device)
    kept = (mass > 0) & ((rank < k) | (k <= 0)) & (mass >= m)
    among = torch.where((rank < k) | (k <= 0), mass, 0.0)
    before = among.cumsum(1)
    kept &= (before - among < p * before[:, -1:]) | (p >= 1)
    kept[:, 0] = True
    w = torch.where(kept, mass, 0.0).cumsum(1)  # from the likeliest token down, ties from the lowest index
    place = torch.where(t > 0, (w <= st["u"].double()[:, None] * w[:, -1:]).sum(1, keepdim=True), 0)
    token = order.gather(1, place)[:, 0]
    if not st["logprob"]:
        return {"token": token}
    # among what was kept; a greedy choice is certain
    gap = (z.gather(1, place) - top) / t
    return {"token": token, "logprob": torch.where(t > 0, gap - w[:, -1:].log(), 0.0)[:, 0].float()}


def run(state):
    op = state["op"]
    if not own:
        return {"norm": _plain_norm, "quant": _plain_quant, "linear": _plain_linear, "sample": _plain_sample}[op](state)
    import mamba3_amd as m
    if op == "norm":
        x, residual, weight = state["x"], state["residual"], state["weight"]
        if state["out"] != "same":
            total, y = m.add_rms_norm_mx(x, residual, weight, state["scale"], _EPS, format=state["out"])
            return {"total": total, "y": y.dequantize()}
        with torch.set_grad_enabled(state["train"]):
            total, y = m.add_rms_norm(x, residual, weight, state["scale"], _EPS)
        if not state["train"]:
            return {"total": total, "y": y}
        dx, dr, dw = torch.autograd.grad([total, y], [x, residual, weight], [state["dtotal"], state["dy"]])
        return {"total": total.detach(), "y": y.detach(), "dx": dx, "dresidual": dr, "dweight": dw}
    if op == "quant":
        q = (m.silu_mul_mx if state["gated"] else m.quantize_mx)(state["x"], format=state["format"])
        return {"values": q.dequantize()}
    if op == "linear":
        x = state["x_in"]
        x = x if torch.is_tensor(x) else m.MXTensor(*x, (state["rows"], state["k"]), state["x"])
        w = m.MXTensor(*state["w"], (state["n"], state["k"]), "e2m1")
        return {"y": m.mx_linear(x, w, state["res"], state["scale"], out_dtype=_TYPES[state["out"]])}
    got = m.sample_tokens(state["logits"], state["u"], state["temperature"], state["top_k"], state["top_p"], state["min_p"], return_logprob=state["logprob"])
    return {"token": got[0], "logprob": got[1]} if state["logprob"] else {"token": got}


def work(case):
    op = case["op"]
    if op == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * _TYPES[case["dtype"]].itemsize + case["rows"] * ((28 if case["each"] else 12) + (4 if case["logprob"] else 0)), "flops": 4 * n}
    if op == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        out = _TYPES[case["out"]].itemsize
        x = _TYPES[case["x"]].itemsize if case["x"] in _TYPES else _BITS[case["x"]] / 8 + 1 / 32
        return {"bytes": m * k * x + n * k * (0.5 + 1 / 32) + m * n * out * (2 if case["residual"] else 1), "flops": 2 * m * k * n}
    size = _TYPES[case["dtype"]].itemsize
    if op == "quant":
        n = case["rows"] * case["k"]
        # the stored form is written and read back: both are what the call is for
        return {"bytes": n * (size * (2 if case["gated"] else 1) + 2 * (_BITS[case["format"]] / 8 + 1 / 32) + 2), "flops": 4 * n}
    n = case["rows"] * case["d"]
    if case["out"] != "same":
        return {"bytes": n * (3 * size + 2 * (1 + 1 / 32) + 2) + case["d"] * size, "flops": 8 * n}
    return {"bytes": n * size * (9 if case["train"] else 4) + case["d"] * size * (2 if case["train"] else 1), "flops": (20 if case["train"] else 6) * n}


# ------------------------------------------------------------------ 64 bits
def _exact_scale(top, fmt):
    """2 to the smallest whole number under which `top` rounds to an element: counted up from below, at least -127."""
    limit = 7.0 if fmt == "e2m1" else 464.0
    e = torch.ceil(torch.log2(top.clamp(min=1e-300) / limit)).clamp(min=-127) - 2
    for _ in range(4):
        s = top / torch.exp2(e)
        e = e + ((s >= limit) if fmt == "e2m1" else (s > limit))
    return torch.exp2(torch.where(top > 0, e.clamp(min=-127), 0))


def _exact_values(x, fmt):
    rows, k = x.shape
    b = F.pad(x, (0, -k % 32)).view(rows, -1, 32)
    scale = _exact_scale(b.abs().amax(-1, keepdim=True), fmt)
    if fmt == "e2m1":
        grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    else:
        grid = torch.arange(127, dtype=torch.uint8, device=x.device).view(torch.float8_e4m3fn).double()
    half = (grid[1:] + grid[:-1]) / 2
    v = b.abs() / scale
    at = torch.searchsorted(half, v)                       # a tie goes down here, and up below where the lower one is odd
    tie = (at < len(half)) & (v == half[at.clamp(max=len(half) - 1)]) & (at % 2 == 1)
    q = torch.copysign(grid[at + tie.long()], b) * scale
    return q.view(rows, -1)[:, :k]


def _exact_held(data, scales, fmt, k):
    if fmt == "e4m3":
        v = data.view(torch.float8_e4m3fn).double()
    else:
        code = torch.empty(data.shape[0], 2 * data.shape[1], dtype=torch.long, device=data.device)
        code[:, 0::2], code[:, 1::2] = data % 16, data // 16
        e, f, s = code // 2 % 4, code % 2, code // 8
        v = torch.where(e > 0, (1 + f / 2) * torch.exp2((e - 1).double()), f / 2) * (1 - 2 * s)
    return (v * torch.exp2(scales.double() - 127).repeat_interleave(32, 1))[:, :k].double()


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        dt = st["x"].dtype
        x, res, w = (st[key].detach().double() for key in ("x", "residual", "weight"))
        total = res + st["scale"] * x
        t = total.to(dt).double().requires_grad_(case["train"])  # the norm is of the sum as it is stored
        w.requires_grad_(case["train"])
        y = F.rms_norm(t, (case["d"],), w, _EPS)
        if case["out"] != "same":
            return {"total": total, "y": _exact_values(y, case["out"])}
        if not case["train"]:
            return {"total": total, "y": y}
        dt_, dw = torch.autograd.grad(y, [t, w], st["dy"].double())
        dt_ = dt_ + st["dtotal"].double()
        return {"total": total, "y": y.detach(), "dx": st["scale"] * dt_, "dresidual": dt_, "dweight": dw}
    if op == "quant":
        x = st["x"].double()
        if case["gated"]:
            x = F.silu(x[:, :case["k"]]) * x[:, case["k"]:]
        return {"values": _exact_values(x, case["format"])}
    if op == "linear":
        x = st["x_in"]
        x = _exact_values(x.double(), "e4m3") if torch.is_tensor(x) else _exact_held(*x, case["x"], case["k"])
        y = F.linear(x, _exact_held(*st["w"], "e2m1", case["k"])) * st["scale"]
        return {"y": y if st["res"] is None else st["res"].double() + y}
    if not case["logprob"]:
        return None  # tokens alone: whole numbers
    logits = st["logits"].double()
    greedy = torch.zeros(case["rows"], dtype=torch.bool, device=logits.device)
    setting = {}
    for key, off in (("top_k", case["vocab"]), ("top_p", 2.0), ("min_p", 0.0), ("temperature", 1.0)):
        v = st[key] if case["each"] else torch.full_like(st["u"], case[key], dtype=torch.float64)
        greedy |= (v <= 0) & (key == "temperature")
        setting[key] = torch.where((v <= 0) if key != "top_p" else (v >= 1), off, v.double())[:, None]
    prob = torch.softmax(logits / setting["temperature"], 1)
    ranked, order = torch.sort(prob, dim=1, descending=True, stable=True)
    count = torch.minimum(setting["top_k"].long(), (ranked >= setting["min_p"] * ranked[:, :1]).sum(1, keepdim=True))
    share = ranked.cumsum(1)
    share = share / share.gather(1, setting["top_k"].long().clamp(max=case["vocab"]) - 1)
    count = torch.minimum(count, 1 + (share < setting["top_p"]).sum(1, keepdim=True)).clamp(min=1, max=case["vocab"])
    left = torch.where(torch.arange(case["vocab"], device=order.device) < count, ranked, 0.0)
    left = left / left.sum(1, keepdim=True)
    at = torch.searchsorted(left.cumsum(1), st["u"].double()[:, None], right=True).clamp(max=case["vocab"] - 1)
    return {"token": None, "logprob": torch.where(greedy, 0.0, left.gather(1, at).log()[:, 0])}
