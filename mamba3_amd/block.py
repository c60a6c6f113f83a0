"""Residual block and language model around KulaMamba: drop-in for mamba3.block
(mamba3/block.py:16-231).

These are the callers of the SSD path (norms, SwiGLU MLP, embedding, tied lm_head,
greedy/sampled decode loop) and run as PyTorch ops; the SSD itself runs in the HIP
kernels through KulaMamba. Module names, registration order and initialisation order
equal the reference's so seeded models hold identical weights.
"""

from __future__ import annotations

import math
import threading
import weakref

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.nn.modules.module import _has_any_global_hook
from torch.utils.checkpoint import checkpoint as grad_checkpoint

from . import _native, ops
from .layer import KulaMamba, RMSNorm
from .loss import linear_cross_entropy
from .mlp import swiglu_mlp
from .mx import MXTensor, mx_linear, quantize_mx
from .sample import sample_tokens


def add_scaled_linear(x: torch.Tensor, lin: nn.Linear, inp: torch.Tensor, scale: float,
                      inplace: bool = False) -> torch.Tensor:
    """x + scale * lin(inp) as one GEMM: the residual x enters hipBLASLt as C with beta = 1
    and the scale as alpha, so the projection's output is neither rounded nor stored before
    the add (the reference runs the projection, the scale and the add as three ops,
    mamba3/block.py:84-91). torch.addmm first copies x into its new output; with inplace
    (x is the caller's own intermediate and no autograd graph needs it) the GEMM accumulates
    into x itself and that copy is saved."""
    inp2 = inp.reshape(-1, inp.shape[-1])
    if inplace and x.is_contiguous():
        x2 = x.view(-1, x.shape[-1])
        x2.addmm_(inp2, lin.weight.t(), beta=1.0, alpha=scale)
        if lin.bias is not None:
            x2.add_(lin.bias, alpha=scale)
        return x
    out = torch.addmm(x.reshape(-1, x.shape[-1]), inp2, lin.weight.t(), beta=1.0, alpha=scale)
    if lin.bias is not None:
        out = out + lin.bias * scale
    return out.view(x.shape)


def _as_written(m: nn.Module, cls: type) -> bool:
    """Calling `m` runs cls.forward and nothing else: no subclass, no forward of its own, no hooks (its own or those of
    all modules)."""
    return (type(m) is cls and "forward" not in m.__dict__
            and not (m._forward_hooks or m._forward_pre_hooks or m._backward_hooks or m._backward_pre_hooks)
            and not _has_any_global_hook())


def _only_weight(lin: nn.Module) -> bool:
    """Calling `lin` is x W^T."""
    return _as_written(lin, nn.Linear) and lin.bias is None


class _MXCopy:
    """The 4-bit copy of some weights, and which weights at which versions. It holds on to their memory, so that an address is not
    another weight's as long as it is compared; their objects are compared too, since a new parameter of the same memory counts
    its versions anew. Copied or pickled it is empty: the other module's weights are others."""

    __slots__ = ("mx", "of", "memory", "streams", "in_graph")

    def __init__(self, *weights: torch.Tensor):
        self.mx = None
        self.of, self.memory = [(weakref.ref(w), w.data_ptr(), w._version, w.dtype) for w in weights], [w.detach() for w in weights]
        self.streams = set()   # that the allocator knows as its readers
        self.in_graph = False  # a captured graph reads it

    def __reduce__(self):
        return _MXCopy, ()

    def is_of(self, weights: tuple[torch.Tensor, ...]) -> bool:
        if len(self.of) != len(weights):
            return False
        for (ref, address, version, dtype), w in zip(self.of, weights):
            if ref() is not w or w._version != version or w.data_ptr() != address or w.dtype != dtype:
                return False
        return True

    def read(self) -> MXTensor:
        """The copy for work on the current stream. Once another has taken its place the allocator keeps its memory until the
        streams that read it have come to that point."""
        mx = self.mx
        known = _native.stream_of(mx.data) in self.streams
        if not (known and self.in_graph) and torch.cuda.is_current_stream_capturing():
            self.in_graph = True
        elif not known:
            stream = torch.cuda.current_stream(mx.device)
            mx.data.record_stream(stream)
            mx.scales.record_stream(stream)
            self.streams.add(_native.stream_of(mx.data))
        return mx

    def release(self) -> None:
        """Waits for graphs that read the copy, whose memory is about to be given back: the allocator does not know their streams."""
        if self.in_graph:
            torch.cuda.synchronize(self.mx.device)


def _mx_copy(owner: nn.Module, *weights: torch.Tensor, anew: bool = False) -> MXTensor:
    """The 4-bit copy of the weights, one below the other, that `owner` keeps: made when first asked for and again after one
    was replaced or changed in place (which their version counters tell) or when asked for `anew`. It goes to memory of its own, so
    that work under way keeps what it reads; where a captured graph reads the old one, into that one's memory behind all work on the
    GPU, so that the graph goes on with the new weights."""
    kept = owner.__dict__.get("_mx")
    if kept is None or anew or not kept.is_of(weights):
        with _MX_LOCK:
            kept = owner.__dict__.get("_mx")
            if kept is None or anew or not kept.is_of(weights):
                kept = owner.__dict__["_mx"] = _mx_made(kept, weights)
    return kept.read()


_MX_LOCK = threading.RLock()  # copies are made by one thread at a time


def _mx_made(kept: _MXCopy | None, weights: tuple[torch.Tensor, ...]) -> _MXCopy:
    """The copy of the weights in the place of `kept`."""
    if any(w.is_inference() for w in weights):
        raise RuntimeError("4-bit weights need parameters that count their changes; those made in torch.inference_mode() do not: make or load "
                           "the model outside of it")
    if weights[0].is_cuda and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("a graph is being captured and the 4-bit weights are not there yet: run the model once before")
    made = _MXCopy(*weights)  # of the versions before they are read
    with torch.inference_mode(False), torch.no_grad():  # copies outlive the mode that they are made in
        mx = quantize_mx(weights[0] if len(weights) == 1 else torch.cat(weights))
        if kept is not None:
            kept.release()
        made.in_graph = kept is not None and kept.in_graph and kept.mx.shape == mx.shape and kept.mx.device == mx.device
        if made.in_graph:
            kept.mx.data.copy_(mx.data)
            kept.mx.scales.copy_(mx.scales)
            mx, made.streams = kept.mx, kept.streams
        else:
            made.streams.add(_native.stream_of(mx.data))  # it was allocated on
    made.mx = mx
    # from here on any stream may read it
    torch.cuda.current_stream(mx.device).synchronize()
    return made


class SwiGLU(nn.Module):
    """w_down(silu(w_gate x) * w_up x) (mamba3/block.py:16-26)."""

    def __init__(self, d_model: int, d_ff: int | None = None, bias: bool = False):
        super().__init__()
        if d_ff is None:
            d_ff = int(d_model * 8 / 3 / 64 + 1) * 64
        self.w_gate = nn.Linear(d_model, d_ff, bias=bias)
        self.w_up = nn.Linear(d_model, d_ff, bias=bias)
        self.w_down = nn.Linear(d_ff, d_model, bias=bias)

    def hidden(self, x: torch.Tensor) -> torch.Tensor:
        """silu(w_gate x) * w_up x: w_down's input. For bf16 without autograd this is one GEMM
        over the concatenated [w_gate; w_up] weight (zero rows pad it to whole 256-column
        tiles; cached per weight version) and one silu * mul pass (m3_silu_mul) instead of
        two GEMMs and two element-wise passes."""
        wg, wu = self.w_gate.weight, self.w_up.weight
        if (torch.is_grad_enabled() or torch.compiler.is_compiling() or x.dtype != torch.bfloat16
                or wg.dtype != torch.bfloat16 or self.w_gate.bias is not None
                or self.w_up.bias is not None or not x.is_cuda):
            return F.silu(self.w_gate(x)) * self.w_up(x)
        d_ff = wg.shape[0]
        key = (wg.data_ptr(), wg._version, wu.data_ptr(), wu._version, wg.device)
        cache = self.__dict__.get("_gate_up")
        if cache is None or cache[0] != key:
            n = 2 * d_ff
            npad = -(-n // 256) * 256 if (-(-n // 256) * 256 - n) * 16 <= n else n
            w = torch.zeros(npad, wg.shape[1], dtype=wg.dtype, device=wg.device)
            w[:d_ff] = wg
            w[d_ff:n] = wu
            cache = (key, w)
            self.__dict__["_gate_up"] = cache
        gu = F.linear(x.reshape(-1, x.shape[-1]), cache[1])
        return ops.silu_mul_fast(gu, d_ff).view(*x.shape[:-1], d_ff)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return self.w_down(self.hidden(x))

    def fusable(self, x: torch.Tensor) -> bool:
        """swiglu_mlp takes these projections and x (one dtype of its two) and computes what calling them would."""
        lins = (self.w_gate, self.w_up, self.w_down)
        return (x.is_cuda and x.dtype in (torch.float32, torch.bfloat16) and not torch.is_autocast_enabled("cuda")
                and _as_written(self, SwiGLU)
                and all(_only_weight(p) and p.weight.dtype == x.dtype and p.weight.device == x.device for p in lins))

    def fused(self, x: torch.Tensor, residual: torch.Tensor | None = None, scale: float = 1.0) -> torch.Tensor:
        """[residual +] scale * w_down(silu(w_gate x) * w_up x) as one operator (swiglu_mlp)."""
        return swiglu_mlp(x, self.w_gate.weight, self.w_up.weight, self.w_down.weight, residual, scale)


class KulaMambaBlock(nn.Module):
    """Pre-norm residual block: x + s*ssm(norm(x)), then x + s*mlp(norm(x))
    (mamba3/block.py:29-107)."""

    def __init__(
        self,
        d_model: int,
        d_state: int = 128,
        expand: int = 2,
        headdim: int = 64,
        ngroups: int | None = None,
        mimo_rank: int = 2,
        chunk_size: int = 64,
        use_mlp: bool = True,
        mlp_expand: float = 2.667,
        norm_eps: float = 1e-5,
        bias: bool = False,
        residual_scale: float = 1.0,
        gradient_checkpointing: bool = False,
        use_trapezoidal: bool = True,
        use_complex_ssm: bool = True,
    ):
        super().__init__()
        self.residual_scale = residual_scale
        self.gradient_checkpointing = gradient_checkpointing
        self.ssm_norm = RMSNorm(d_model, eps=norm_eps)
        self.ssm = KulaMamba(
            d_model=d_model, d_state=d_state, expand=expand, headdim=headdim,
            ngroups=ngroups, mimo_rank=mimo_rank, chunk_size=chunk_size, bias=bias,
            use_trapezoidal=use_trapezoidal, use_complex_ssm=use_complex_ssm,
        )
        self.use_mlp = use_mlp
        if use_mlp:
            d_ff = int(d_model * mlp_expand / 64 + 1) * 64
            self.mlp_norm = RMSNorm(d_model, eps=norm_eps)
            self.mlp = SwiGLU(d_model, d_ff, bias=bias)

    # Run the MLP and its residual as one operator (swiglu_mlp: forward and backward on kernels of
    # this package) instead of library products around element-wise passes. Off by default: its
    # roundings differ (g, u and, in the backward, dh are not rounded to bf16).
    fused_mlp: bool = False

    # Without gradients, multiply by 4-bit copies of the weights (KulaMambaLM.quantize_mx). Off by default.
    mx_weights: bool = False

    def _mx_projections(self, anew: bool = False) -> tuple[MXTensor, ...]:
        """in_proj, out_proj and with an MLP [w_gate; w_up] and w_down in 4 bits."""
        lins = [self.ssm.in_proj, self.ssm.out_proj]
        whole = isinstance(self.ssm, KulaMamba) and _as_written(self.ssm_norm, RMSNorm) and self.ssm_norm.dim == -1
        if self.use_mlp:
            mlp = self.mlp
            whole = whole and _as_written(mlp, SwiGLU) and _as_written(self.mlp_norm, RMSNorm) and self.mlp_norm.dim == -1
            if whole:
                lins += [mlp.w_gate, mlp.w_up, mlp.w_down]
        if not whole or not all(_only_weight(lin) for lin in lins):
            raise RuntimeError("4-bit weights need projections without bias and norms of the last dimension, without hooks or forwards of "
                               "their own")
        w = [lin.weight for lin in lins]
        copies = (_mx_copy(lins[0], w[0], anew=anew), _mx_copy(lins[1], w[1], anew=anew))
        return copies if not self.use_mlp else (*copies, _mx_copy(self.mlp, w[2], w[3], anew=anew), _mx_copy(lins[4], w[4], anew=anew))

    def _mx_on(self) -> bool:
        return self.mx_weights and not torch.is_grad_enabled()

    @torch.compiler.disable
    def _mx_block(self, x: torch.Tensor, ssd):
        """The block on 4-bit weights: what is normed, gated and given out by the SSD is rounded to 8 bits as the next product's
        input, the residual stays in x's type. ssd: in_proj's output -> (out_proj's input, state)."""
        w, s = self._mx_projections(), self.residual_scale
        y, state = ssd(mx_linear(x, w[0], norm_weight=self.ssm_norm.weight, eps=self.ssm_norm.eps))
        x = mx_linear(y.view(*x.shape[:-1], -1), w[1], x, s)
        if self.use_mlp:
            gate_up = mx_linear(x, w[2], norm_weight=self.mlp_norm.weight, eps=self.mlp_norm.eps)
            x = mx_linear(gate_up, w[3], x, s, gated=True)
        return x, state

    def _ssm_forward(self, x_normed):
        return self.ssm(x_normed)

    def _mlp_forward(self, x_normed):
        if self.fused_mlp and self.mlp.fusable(x_normed):
            return self.mlp.fused(x_normed)
        return self.mlp(x_normed)

    # The residual adds run as the beta = 1 input of the out_proj / w_down GEMMs
    # (add_scaled_linear); with gradient checkpointing the branches are recomputed whole.
    def forward(self, x: torch.Tensor, _own_input: bool = False) -> torch.Tensor:
        """_own_input (internal): x is an intermediate of the caller's forward
        (KulaMambaLM), so without autograd the first residual add may overwrite it. The
        second add overwrites the first one's output whenever no autograd graph needs it."""
        if self._mx_on():
            self.ssm._check_sequence(x)
            return self._mx_block(x, self.ssm.ssd_from_proj)[0]
        ckpt = self.gradient_checkpointing and self.training
        nograd = not torch.is_grad_enabled()
        if ckpt:
            h = grad_checkpoint(self._ssm_forward, self.ssm_norm(x), use_reentrant=False)
            x = x + h * self.residual_scale
        else:
            y, _ = self.ssm._pre_out(self.ssm_norm(x))
            x = add_scaled_linear(x, self.ssm.out_proj, y, self.residual_scale,
                                  inplace=_own_input and nograd)
        if self.use_mlp:
            if ckpt:
                m = grad_checkpoint(self._mlp_forward, self.mlp_norm(x), use_reentrant=False)
                x = x + m * self.residual_scale
            else:
                x = self._mlp_residual(x, inplace=nograd)
        return x

    def _mlp_residual(self, x: torch.Tensor, inplace: bool = False) -> torch.Tensor:
        n = self.mlp_norm(x)
        if self.fused_mlp and n.dtype == x.dtype and self.mlp.fusable(n):
            return self.mlp.fused(n, x, self.residual_scale)
        return add_scaled_linear(x, self.mlp.w_down, self.mlp.hidden(n), self.residual_scale, inplace=inplace)

    def _small_step_usable(self, x: torch.Tensor) -> bool:
        """The decode step runs on the small-batch projection kernels (norm + in_proj,
        out_proj + residual, norm + SwiGLU, w_down + residual): bf16, at most 8 rows, no
        biases, last-dimension norms, nothing to differentiate."""
        m = x.shape[0]
        if m > _native.SMALL_PROJ_MAX_ROWS or x.dtype != torch.bfloat16:
            return False
        ssm, norm = self.ssm, self.ssm_norm
        ip, op = ssm.in_proj, ssm.out_proj
        # every projection's K: d_model (with a norm), d_inner, d_ff
        if not (_native.small_proj_ok(m, op.in_features) and ip.bias is None and op.bias is None
                and norm.dim in (-1, 1)):
            return False
        if not self.use_mlp:
            return ops.small_proj_usable(x, norm.weight, ip.weight, op.weight, norm=True)
        mlp, norm2 = self.mlp, self.mlp_norm
        gate, up, down = mlp.w_gate, mlp.w_up, mlp.w_down
        return (_native.small_proj_ok(m, down.in_features) and gate.bias is None
                and up.bias is None and down.bias is None and norm2.dim in (-1, 1)
                and ops.small_proj_usable(x, norm.weight, ip.weight, op.weight, norm2.weight,
                                          gate.weight, up.weight, down.weight, norm=True))

    def _small_step_tail(self, x: torch.Tensor, y: torch.Tensor) -> torch.Tensor:
        """x + s out_proj(y), then the MLP residual, on the small-batch kernels."""
        s = self.residual_scale
        x = ops.small_linear_fast(y, None, 0.0, self.ssm.out_proj.weight, x, s)
        if self.use_mlp:
            mlp = self.mlp
            h = ops.small_swiglu_fast(x, self.mlp_norm.weight, float(self.mlp_norm.eps),
                                 mlp.w_gate.weight, mlp.w_up.weight)
            x = ops.small_linear_fast(h, None, 0.0, mlp.w_down.weight, x, s)
        return x

    def step(self, x: torch.Tensor, ssm_state: dict):
        if self._mx_on():
            y, state = self._mx_block(self.ssm._check_token(x), lambda proj: self.ssm._step_from_proj(proj, ssm_state))
            return y.view(x.shape), state
        if self._small_step_usable(x):
            proj = ops.small_linear_fast(x, self.ssm_norm.weight, float(self.ssm_norm.eps),
                                    self.ssm.in_proj.weight, None, 1.0)
            y, new_state = self.ssm._step_from_proj(proj, ssm_state)
            return self._small_step_tail(x, y), new_state
        y, new_state = self.ssm._step_pre_out(self.ssm_norm(x), ssm_state)
        x = add_scaled_linear(x, self.ssm.out_proj, y.view(*x.shape[:-1], -1), self.residual_scale)
        if self.use_mlp:
            x = self._mlp_residual(x, inplace=not torch.is_grad_enabled())
        return x, new_state

    def prefill(self, x: torch.Tensor, _own_input: bool = False):
        """_own_input as in forward."""
        if self._mx_on():
            self.ssm._check_sequence(x)
            return self._mx_block(x, lambda proj: self.ssm.ssd_from_proj(proj, return_state=True))
        nograd = not torch.is_grad_enabled()
        y, state = self.ssm._pre_out(self.ssm_norm(x), return_state=True)
        x = add_scaled_linear(x, self.ssm.out_proj, y, self.residual_scale,
                              inplace=_own_input and nograd)
        if self.use_mlp:
            x = self._mlp_residual(x, inplace=nograd)
        return x, state


class KulaMambaLM(nn.Module):
    """Embedding -> n_layers KulaMambaBlock -> RMSNorm -> (tied) lm_head
    (mamba3/block.py:110-231)."""

    def __init__(
        self,
        vocab_size: int,
        d_model: int = 768,
        n_layers: int = 12,
        d_state: int = 128,
        expand: int = 2,
        headdim: int = 64,
        ngroups: int | None = None,
        mimo_rank: int = 2,
        chunk_size: int = 64,
        use_mlp: bool = True,
        tie_weights: bool = True,
        norm_eps: float = 1e-5,
        bias: bool = False,
        residual_scale: str = "depth",
        gradient_checkpointing: bool = False,
        use_trapezoidal: bool = True,
        use_complex_ssm: bool = True,
    ):
        super().__init__()
        self.d_model = d_model
        self.n_layers = n_layers
        scale = 1.0 / math.sqrt(2 * n_layers) if residual_scale == "depth" else 1.0
        self.embedding = nn.Embedding(vocab_size, d_model)
        self.layers = nn.ModuleList([
            KulaMambaBlock(
                d_model=d_model, d_state=d_state, expand=expand, headdim=headdim,
                ngroups=ngroups, mimo_rank=mimo_rank, chunk_size=chunk_size, use_mlp=use_mlp,
                norm_eps=norm_eps, bias=bias, residual_scale=scale,
                gradient_checkpointing=gradient_checkpointing,
                use_trapezoidal=use_trapezoidal, use_complex_ssm=use_complex_ssm,
            )
            for _ in range(n_layers)
        ])
        self.norm = RMSNorm(d_model, eps=norm_eps)
        self.lm_head = nn.Linear(d_model, vocab_size, bias=False)
        if tie_weights:
            self.lm_head.weight = self.embedding.weight
        self._init_weights()

    def _init_weights(self) -> None:
        """N(0, 0.02) for the embedding and every Linear except the (tied) head, then the
        KulaMamba-specific re-initialisation (mamba3/block.py:166-176)."""
        nn.init.normal_(self.embedding.weight, std=0.02)
        for m in self.modules():
            if isinstance(m, nn.Linear) and m is not self.lm_head:
                nn.init.normal_(m.weight, std=0.02)
                if m.bias is not None:
                    nn.init.zeros_(m.bias)
        for m in self.modules():
            if isinstance(m, KulaMamba):
                m._init_weights(dt_min=0.001, dt_max=0.1)

    def fuse_mlp(self, on: bool = True) -> "KulaMambaLM":
        """Switches every block's MLP to the fused operator (KulaMambaBlock.fused_mlp) or back."""
        for layer in self.layers:
            layer.fused_mlp = on
        return self

    # Without gradients, multiply by 4-bit copies of the weights (quantize_mx). Off by default.
    mx_weights: bool = False

    def quantize_mx(self, on: bool = True) -> "KulaMambaLM":
        """Switches products without gradients (generate, and forward, loss, prefill and step under torch.no_grad()) to 4-bit
        copies of the weights and activations in 8 bits, both microscaled (quantize_mx, mx_linear), or back and frees
        the copies: graphs captured with them are not to be replayed after that. Gradients and the embedding use the weights
        themselves, which stay. A copy is made anew when the model runs and its weight was replaced or changed in place; after changes
        that leave no trace (through `.data`, or by a graph's replay, as of a captured optimizer step), call this again. Copies that
        captured graphs read stay in their memory, behind all work on the GPU, and others go to new memory. Weights made in torch.inference_mode() count no changes and are
        refused. Needs projections without bias. A block inside a reentrant checkpoint runs its forward without gradients: switch
        back before training with one."""
        if on:
            try:
                for layer in self.layers:
                    layer._mx_projections(anew=True)
                self._mx_head(anew=True)
            except Exception:
                if not self.mx_weights:
                    self.quantize_mx(False)
                raise
        else:
            for m in self.modules():
                kept = m.__dict__.pop("_mx", None)
                if kept is not None:
                    kept.release()
        self.mx_weights = on
        for layer in self.layers:
            layer.mx_weights = on
        return self

    def _mx_on(self) -> bool:
        return self.mx_weights and not torch.is_grad_enabled()

    def _mx_head(self, anew: bool = False) -> MXTensor:
        if not (_only_weight(self.lm_head) and _as_written(self.norm, RMSNorm) and self.norm.dim == -1):
            raise RuntimeError("4-bit weights need a head without bias and a norm of the last dimension, without hooks or forwards of their own")
        return _mx_copy(self.lm_head, self.lm_head.weight, anew=anew)

    @torch.compiler.disable
    def _mx_logits(self, x: torch.Tensor) -> torch.Tensor:
        return mx_linear(x, self._mx_head(), norm_weight=self.norm.weight, eps=self.norm.eps)

    def loss(self, input_ids: torch.Tensor, labels: torch.Tensor, ignore_index: int = -100) -> torch.Tensor:
        """The mean next-token cross entropy that forward returns as "loss" (fp32), without the
        logits: the head and the loss are one operator (linear_cross_entropy), so a training step
        holds neither the (tokens, vocab) logits nor their gradient. A head that is more than its weight
        (a bias, hooks, a subclass) is called, and its logits kept. labels: (B, T), position t is
        predicted from t - 1; those equal to ignore_index do not count."""
        if labels.shape != input_ids.shape:
            raise ValueError(f"labels have shape {tuple(labels.shape)}, expected {tuple(input_ids.shape)}")
        x = self.embedding(input_ids)
        for layer in self.layers:
            x = layer(x, _own_input=True)
        # the last position predicts nothing: it is ignored rather than cut off, which would copy
        # the hidden states
        target = torch.full_like(labels, ignore_index)
        target[:, :-1] = labels[:, 1:]
        if self._mx_on():
            return F.cross_entropy(self._mx_logits(x).flatten(0, -2).float(), target.flatten(), ignore_index=ignore_index)
        x = self.norm(x)
        if not _only_weight(self.lm_head):
            return F.cross_entropy(self.lm_head(x).flatten(0, -2).float(), target.flatten(), ignore_index=ignore_index)
        return linear_cross_entropy(x, self.lm_head.weight, target, ignore_index)

    def forward(self, input_ids: torch.Tensor, labels: torch.Tensor | None = None) -> dict:
        x = self.embedding(input_ids)
        for layer in self.layers:
            x = layer(x, _own_input=True)
        logits = self._mx_logits(x) if self._mx_on() else self.lm_head(self.norm(x))
        result = {"logits": logits}
        if labels is not None:
            pred = logits[:, :-1].contiguous()
            tgt = labels[:, 1:].contiguous()
            result["loss"] = F.cross_entropy(pred.view(-1, pred.size(-1)), tgt.view(-1))
        return result

    # Replay the per-token decode step (embedding, every block's step, norm, lm_head) as one
    # captured HIP graph instead of launching each op from Python. Sampling stays eager.
    decode_graph: bool = True

    @torch.no_grad()
    def generate(self, input_ids: torch.Tensor, max_new_tokens: int = 100,
                 temperature: float = 1.0, top_k: int | None = None, top_p: float | None = None,
                 min_p: float | None = None, generator: torch.Generator | None = None) -> torch.Tensor:
        """Parallel prefill of the prompt, then one `step` per new token
        (mamba3/block.py:195-231). temperature=0 is greedy argmax.

        With top_p, min_p or a generator (of the ids' device) tokens are drawn by sample_tokens from one random number a row, else
        with torch.multinomial. There, a row whose logits are all NaN or -inf gives -1 and goes on with token 0; top_k keeps
        exactly as many, ties from the lowest index."""
        own = top_p is not None or min_p is not None or generator is not None
        if own:
            top_p, min_p = 1.0 if top_p is None else float(top_p), 0.0 if min_p is None else float(min_p)
            if not (0.0 <= top_p <= 1.0 and 0.0 <= min_p <= 1.0 and temperature >= 0.0 and (top_k is None or top_k > 0)):
                raise ValueError(f"need top_p and min_p in [0, 1], temperature of at least 0 and top_k of at least 1, got {top_p}, {min_p}, "
                                 f"{temperature} and {top_k}")
        x = self.embedding(input_ids)
        states = []
        for layer in self.layers:
            x, st = layer.prefill(x, _own_input=True)
            states.append(st)
        logits = self._mx_logits(x[:, -1]) if self._mx_on() else self.lm_head(self.norm(x)[:, -1])
        out = [input_ids]
        graph = None
        if self.decode_graph and max_new_tokens > 1 and input_ids.is_cuda:
            graph = _DecodeGraph(self, states, input_ids.shape[0])
        for _ in range(max_new_tokens):
            if own:
                u = torch.rand(logits.shape[0], device=logits.device, generator=generator)
                nxt = sample_tokens(logits, u, temperature, top_k or 0, top_p, min_p).unsqueeze(1)
                out.append(nxt)
                logits = self._next_logits(nxt.squeeze(1).clamp(min=0), states, graph)
                continue
            scores = logits / temperature if temperature > 0 else logits
            if top_k is not None:
                kth = torch.topk(scores, min(top_k, scores.size(-1))).values[:, -1:]
                scores = scores.masked_fill(scores < kth, float("-inf"))
            if temperature > 0:
                nxt = torch.multinomial(F.softmax(scores, dim=-1), num_samples=1)
            else:
                nxt = scores.argmax(dim=-1, keepdim=True)
            out.append(nxt)
            logits = self._next_logits(nxt.squeeze(1), states, graph)
        return torch.cat(out, dim=1)

    def _next_logits(self, tokens: torch.Tensor, states: list, graph: "_DecodeGraph | None") -> torch.Tensor:
        """One step of decoding; without a graph `states` are replaced by the new ones."""
        if graph is not None:
            return graph(tokens)
        x = self.embedding(tokens)
        for i, layer in enumerate(self.layers):
            x, states[i] = layer.step(x, states[i])
        return _lm_logits(self, x)


def _block_step_into(block: KulaMambaBlock, x: torch.Tensor, st_in: dict, st_out: dict):
    """KulaMambaBlock.step (mamba3/block.py:94-100) with the SSM step written into the
    caller's state buffers `st_out` (which must not alias `st_in`)."""
    ssm = block.ssm

    def step(proj):
        y = torch.empty(x.shape[0], ssm.d_inner, device=x.device, dtype=proj.dtype)
        ops.step_into(proj, *ssm._small_params(), None, st_in["h"], st_in["prev_BX"],
                      st_in["angle"], y, st_out["h"], st_out["prev_BX"], st_out["angle"],
                      *ops.layer_args(ssm))
        return y

    if block._mx_on():
        return block._mx_block(x, lambda proj: (step(proj), None))[0]
    small = block._small_step_usable(x)
    if small:
        proj = ops.small_linear_fast(x, block.ssm_norm.weight, float(block.ssm_norm.eps),
                                ssm.in_proj.weight, None, 1.0)
    else:
        proj = ssm.in_proj(block.ssm_norm(x))
    y = step(proj)
    if small:
        return block._small_step_tail(x, y)
    x = add_scaled_linear(x, ssm.out_proj, y, block.residual_scale)
    if block.use_mlp:
        x = block._mlp_residual(x)
    return x


def _lm_logits(lm: "KulaMambaLM", x: torch.Tensor) -> torch.Tensor:
    """lm_head(norm(x)) for decode rows x (B, d_model): one small-batch kernel (norm in its
    prologue) when it applies (mamba3/block.py:182-183)."""
    if lm._mx_on():
        return lm._mx_logits(x)
    w = lm.lm_head.weight
    if (lm.lm_head.bias is None and lm.norm.dim in (-1, 1)
            and ops.small_proj_usable(x, lm.norm.weight, w, norm=True)):
        return ops.small_linear_fast(x, lm.norm.weight, float(lm.norm.eps), w, None, 1.0)
    return lm.lm_head(lm.norm(x))


class _DecodeGraph:
    """One decode step of a KulaMambaLM captured as HIP graphs (torch.cuda.CUDAGraph):
    token ids -> embedding -> every block's step -> norm -> lm_head logits. The decode
    state lives in two static buffer sets; graph 0 reads set 0 and writes set 1, graph 1
    the reverse, and replays alternate between them, so no state is copied. Outputs are
    bitwise those of the eager step (same kernels, same order)."""

    def __init__(self, lm: KulaMambaLM, states: list, batch: int):
        dev = lm.embedding.weight.device
        self.tok = torch.zeros(batch, dtype=torch.long, device=dev)
        self.bufs = [[{k: v.clone() for k, v in st.items()} for st in states],
                     [{k: torch.empty_like(v) for k, v in st.items()} for st in states]]

        def step(src: int):
            x = lm.embedding(self.tok)
            for i, block in enumerate(lm.layers):
                x = _block_step_into(block, x, self.bufs[src][i], self.bufs[1 - src][i])
            return _lm_logits(lm, x)

        # Warm up outside the capture on a side stream (allocator and library handles);
        # it reads set 0 and writes set 1, which the first replay rewrites.
        side = torch.cuda.Stream(device=dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):
            step(0)
        torch.cuda.current_stream(dev).wait_stream(side)
        self.graphs, self.logits = [], []
        for src in (0, 1):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                self.logits.append(step(src))
            self.graphs.append(g)
        torch.cuda.synchronize(dev)
        self.phase = 0

    def __call__(self, tok: torch.Tensor) -> torch.Tensor:
        self.tok.copy_(tok)
        self.graphs[self.phase].replay()
        out = self.logits[self.phase]
        self.phase ^= 1
        return out
