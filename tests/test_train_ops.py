"""Refusals of the training operators (gated MLP, linear cross entropy, gradient clipping), on the
host: nothing here launches a kernel."""

from __future__ import annotations

import ctypes
import math
import random

import pytest
import torch

import mamba3_amd
from mamba3_amd import _native
from mamba3_amd.clip import _refuse_shared_memory

FAKE = 1 << 12  # an address that is never dereferenced: the call is refused first


@pytest.fixture(scope="module")
def lib():
    if not _native.LIB_PATH.exists():
        from mamba3_amd import build
        build.build(verbose=False)
    return _native.lib()


def _size(fn, *args):
    n = ctypes.c_size_t(0)
    return fn(*args, ctypes.byref(n)), n.value


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("rows,d,ff", [(1, 1, 1), (7, 33, 65), (8192, 768, 2112), (1 << 20, 2048, 5504)])
def test_swiglu_sizes_cover_what_is_kept(lib, dtype, rows, d, ff):
    st, saved = _size(lib.m3_swiglu_mlp_saved_size, rows, d, ff, dtype)
    size = 2 if dtype else 4
    # gate and up (24 bits each, or fp32) and h
    assert st == 0 and saved >= rows * ff * ((6 + 2) if dtype else (8 + 4)) and saved % 256 == 0
    st, kept = _size(lib.m3_swiglu_mlp_fwd_workspace_size, rows, d, ff, dtype, 1)
    assert st == 0
    st, alone = _size(lib.m3_swiglu_mlp_fwd_workspace_size, rows, d, ff, dtype, 0)
    assert st == 0 and alone >= kept + rows * ff * size
    st, back = _size(lib.m3_swiglu_mlp_bwd_workspace_size, rows, d, ff, dtype)
    assert st == 0 and back >= 2 * rows * ff * size


def test_swiglu_refuses_bad_arguments(lib):
    def fwd(rows=4, d=64, ff=128, dtype=1, x=FAKE, wg=FAKE, wu=FAKE, wd=FAKE, res=None, y=FAKE, saved=None,
            ws=FAKE, n=1 << 40):
        return lib.m3_swiglu_mlp_fwd(rows, d, ff, dtype, x, wg, wu, wd, res, 1.0, y, saved, ws, n, None)

    for name in ("x", "wg", "wu", "wd", "y"):
        assert fwd(**{name: None}) == 1
    assert fwd(rows=0) == 2 and fwd(d=0) == 2 and fwd(ff=-1) == 2
    assert fwd(rows=(1 << 30) + 1) == 3 and fwd(d=(1 << 20) + 1) == 3 and fwd(ff=(1 << 20) + 1) == 3
    assert fwd(dtype=2) == 3
    for name in ("x", "wg", "wu", "wd", "ws"):
        assert fwd(**{name: FAKE + 8}) == 5
    assert fwd(saved=FAKE + 16) == 5
    assert fwd(ws=None) == 4 and fwd(n=16) == 4

    def bwd(rows=4, dtype=1, x=FAKE, saved=FAKE, dy=FAKE, ws=FAKE, n=1 << 40):
        return lib.m3_swiglu_mlp_bwd(rows, 64, 128, dtype, x, FAKE, FAKE, FAKE, 1.0, saved, dy, FAKE, FAKE, FAKE,
                                     FAKE, ws, n, None)

    assert bwd(x=None) == 1 and bwd(saved=None) == 1 and bwd(dy=None) == 1
    assert bwd(rows=-1) == 2 and bwd(dtype=7) == 3
    assert bwd(dy=FAKE + 2) == 5 and bwd(saved=FAKE + 16) == 5 and bwd(n=0) == 4


def test_xent_refuses_bad_arguments(lib):
    def fwd(rows=4, d=64, vocab=100, dtype=1, red=1, h=FAKE, w=FAKE, t=FAKE, loss=FAKE, lse=FAKE, count=FAKE,
            ws=FAKE, n=1 << 40):
        return lib.m3_linear_xent_fwd(rows, d, vocab, dtype, red, h, w, t, -100, loss, lse, count, ws, n, None)

    for name in ("h", "w", "t", "loss", "lse", "count"):
        assert fwd(**{name: None}) == 1
    assert fwd(rows=0) == 2 and fwd(vocab=0) == 2 and fwd(red=3) == 2 and fwd(red=-1) == 2
    assert fwd(dtype=2) == 3 and fwd(vocab=(1 << 30) + 1) == 3 and fwd(d=(1 << 20) + 1) == 3
    assert fwd(h=FAKE + 8) == 5 and fwd(w=FAKE + 8) == 5 and fwd(ws=None) == 4 and fwd(n=100) == 4

    def bwd(rows=4, red=1, grad=FAKE, dh=FAKE, dw=FAKE, n=1 << 40):
        return lib.m3_linear_xent_bwd(rows, 64, 100, 1, red, FAKE, FAKE, FAKE, -100, FAKE, FAKE, grad, dh, dw, FAKE,
                                      n, None)

    assert bwd(grad=None) == 1 and bwd(rows=0) == 2 and bwd(red=9) == 2 and bwd(n=0) == 4
    assert bwd(dh=None, dw=None) == 0  # nothing asked for, nothing launched


def test_xent_backward_holds_one_piece_of_the_vocabulary(lib):
    st, n = _size(lib.m3_linear_xent_bwd_workspace_size, 8192, 768, 128000, 1, 1, 1)
    # far below the 2.1 GB of bf16 logits: a piece of at most 256 MiB, hidden, fp32 sums
    assert st == 0 and (256 << 20) < n < (1 << 30)


def test_clip_refuses_bad_arguments(lib):
    i64, i32 = ctypes.c_int64, ctypes.c_int32

    def clip(ptrs=(FAKE,), numel=(8,), dtype=(0,), kind=0, norm=FAKE, ws=FAKE, nbytes=1 << 30, n=None):
        n = len(ptrs) if n is None else n
        return lib.m3_clip_grad_norm(n, (ctypes.c_void_p * len(ptrs))(*ptrs), (i64 * len(numel))(*numel),
                                     (i32 * len(dtype))(*dtype), kind, 1, 1.0, norm, ws, nbytes, None)

    assert clip(norm=None) == 1 and clip(ptrs=(None,)) == 1
    assert clip(n=-1) == 2 and clip(numel=(-1,)) == 2
    assert clip(dtype=(5,)) == 3 and clip(kind=2) == 3 and clip(numel=((1 << 36) + 1,)) == 3
    assert clip(ptrs=(FAKE + 2,)) == 5 and clip(ptrs=(FAKE + 1,), dtype=(1,)) == 5
    assert clip(ws=None) == 4 and clip(nbytes=8) == 4 and clip(ws=FAKE + 64) == 5
    assert lib.m3_clip_grad_norm(1, None, None, None, 0, 1, 1.0, FAKE, FAKE, 1 << 30, None) == 1


def _weights(d=8, ff=16, dtype=torch.float32):
    return torch.ones(ff, d, dtype=dtype), torch.ones(ff, d, dtype=dtype), torch.ones(d, ff, dtype=dtype)


def test_swiglu_mlp_refuses():
    wg, wu, wd = _weights()
    x = torch.ones(3, 8)
    with pytest.raises(RuntimeError, match="GPU"):
        mamba3_amd.swiglu_mlp(x, wg, wu, wd)
    with pytest.raises(ValueError, match="do not fit"):
        mamba3_amd.swiglu_mlp(torch.ones(3, 9), wg, wu, wd)
    with pytest.raises(ValueError, match="do not fit"):
        mamba3_amd.swiglu_mlp(x, wg, wu, wd.t())
    with pytest.raises(ValueError, match="two-dimensional"):
        mamba3_amd.swiglu_mlp(x, wg[0], wu, wd)
    with pytest.raises(ValueError, match="residual"):
        mamba3_amd.swiglu_mlp(x, wg, wu, wd, residual=torch.ones(1, 8))
    with pytest.raises(TypeError, match="one dtype"):
        mamba3_amd.swiglu_mlp(x.bfloat16(), wg, wu, wd)
    with pytest.raises(TypeError, match="float32 and bfloat16"):
        mamba3_amd.swiglu_mlp(x.half(), wg.half(), wu.half(), wd.half())


def test_linear_cross_entropy_refuses():
    h, w, t = torch.ones(3, 8), torch.ones(11, 8), torch.zeros(3, dtype=torch.long)
    with pytest.raises(RuntimeError, match="GPU"):
        mamba3_amd.linear_cross_entropy(h, w, t)
    with pytest.raises(ValueError, match="do not fit"):
        mamba3_amd.linear_cross_entropy(h, w.t(), t)
    with pytest.raises(ValueError, match="target has shape"):
        mamba3_amd.linear_cross_entropy(h, w, t[:2])
    with pytest.raises(TypeError, match="int64"):
        mamba3_amd.linear_cross_entropy(h, w, t.int())
    with pytest.raises(ValueError, match="reduction"):
        mamba3_amd.linear_cross_entropy(h, w, t, reduction="median")
    with pytest.raises(TypeError, match="one dtype"):
        mamba3_amd.linear_cross_entropy(h.bfloat16(), w, t)


def test_clip_grad_norm_refuses():
    p = torch.nn.Parameter(torch.ones(4))
    assert mamba3_amd.clip_grad_norm_([p], 1.0).item() == 0.0  # no gradient, nothing to do
    p.grad = torch.ones(4)
    with pytest.raises(RuntimeError, match="GPU"):
        mamba3_amd.clip_grad_norm_([p], 1.0)
    for bad in (1.0, 0.0, math.nan):
        with pytest.raises(ValueError, match="norm_type"):
            mamba3_amd.clip_grad_norm_(p, 1.0, norm_type=bad)
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            mamba3_amd.clip_grad_norm_(p, bad)
    p.grad = torch.ones(4).to_sparse()
    with pytest.raises(TypeError, match="dense"):
        mamba3_amd.clip_grad_norm_(p, 1.0)
    q = torch.nn.Parameter(torch.ones(4, dtype=torch.float16))
    q.grad = torch.ones(4, dtype=torch.float16)
    with pytest.raises(TypeError, match="float32 and bfloat16"):
        mamba3_amd.clip_grad_norm_(q, 1.0)


def test_new_names_are_attributes_beside_the_eight():
    for name in ("swiglu_mlp", "linear_cross_entropy", "clip_grad_norm_"):
        assert callable(getattr(mamba3_amd, name)) and name not in mamba3_amd.__all__


def _elements(g, base):
    """Byte addresses of g's elements from base, each size of them."""
    at = torch.zeros((), dtype=torch.long)
    for k, (n, s) in enumerate(zip(g.shape, g.stride())):
        at = at + (torch.arange(n) * s).view([-1 if i == k else 1 for i in range(g.dim())])
    first = (at.flatten() * g.element_size() + g.data_ptr() - base)[:, None]
    return (first + torch.arange(g.element_size())).flatten()


def test_clip_finds_shared_memory_of_strided_gradients():
    """The host's answer against every byte written down, for small strided views of one buffer in two types."""
    rng = random.Random(0)
    fp32 = torch.zeros(20000)
    bf16 = fp32.view(torch.bfloat16)
    seen = [0, 0]
    for _ in range(1500):
        grads = []
        for _ in range(rng.randint(1, 3)):
            base, dims = rng.choice([fp32, fp32, bf16]), rng.randint(1, 3)
            shape = [rng.randint(1, 9) for _ in range(dims)]
            if rng.random() < 0.5:
                strides = [rng.randint(1, 30) for _ in range(dims)]
            else:  # the axes of one array, in any order
                strides, step = [], rng.choice([1, 2, 3])
                for n in shape:
                    strides.append(step)
                    step *= n + rng.randint(0, 2)
                rng.shuffle(strides)
            grads.append(base.as_strided(shape, strides, rng.randint(0, 120)))
        used = [_elements(g, fp32.data_ptr()) for g in grads]
        shared = torch.cat(used).bincount().max().item() > 1
        whole = [u for g, u in zip(grads, used) if g.is_contiguous()]
        if whole and torch.cat(whole).bincount().max().item() > 1:
            continue  # contiguous ones are compared by the library
        seen[shared] += 1
        if shared:
            with pytest.raises(ValueError, match="overlap|share memory"):
                _refuse_shared_memory(grads)
        else:
            _refuse_shared_memory(grads)
    assert min(seen) > 200


def test_clip_tells_large_strided_gradients_apart():
    """Slices of a weight of 100 M elements, which is never touched: answered from the strides."""
    flat = torch.empty(8192 * 12288)
    m = flat.view(8192, 12288)
    for grads in ((m[:, :4096], m[:, 4096:8192], m[:, 8192:]), (flat[::3], flat[1::3]), (flat[::6], flat[1::2]),
                  (m[:4096].t(), m[4096:]), (m.view(64, 128, 96, 128)[:, :, ::2], m.view(64, 128, 96, 128)[:, :, 1::2, 5:])):
        _refuse_shared_memory(list(grads))
    for grads in ((m[:, :4097], m[:, 4096:8192]), (flat[::7], flat[3::11]), (m.t(), m[8191:]), (flat.as_strided((100, 100), (99, 1)),)):
        with pytest.raises(ValueError, match="overlap|share memory"):
            _refuse_shared_memory(list(grads))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_swiglu_saved_size_in_python_equals_the_librarys(lib, dtype):
    for rows in (1, 2, 15, 16, 17, 300, 777, 4096, 8193, (1 << 20) + 3):
        for ff in (1, 3, 4, 7, 8, 9, 15, 16, 17, 65, 320, 1363, 2112, 5504):
            st, n = _size(lib.m3_swiglu_mlp_saved_size, rows, 64, ff, _native.dtype_code(dtype))
            assert st == 0 and n == _native.swiglu_mlp_saved_bytes(rows, ff, dtype), (rows, ff)


def test_swiglu_traces_with_symbolic_sizes():
    """The ops' fake kernels keep sizes symbolic: no guard says what they are, so one trace serves all row counts."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from mamba3_amd import ops

    def step(x, wg, wd):
        y, saved = ops.swiglu_mlp(x, wg, wg, wd, None, 1.0, True)
        return ops.swiglu_mlp_bwd(x, wg, wg, wd, 1.0, saved, y, [True, False, True, True])

    bf16 = torch.bfloat16
    env = make_fx(step, tracing_mode="symbolic")(torch.empty(300, 128, dtype=bf16), torch.empty(320, 128, dtype=bf16),
                                                 torch.empty(128, 320, dtype=bf16)).shape_env
    assert not env.replacements and not env.guards

    def loss(hidden, weight, target):
        out, lse, count = ops.linear_xent(hidden, weight, target, -100, 1)
        return ops.linear_xent_bwd(hidden, weight, target, -100, 1, lse, count, out, [True, True])

    env = make_fx(loss, tracing_mode="symbolic")(torch.empty(300, 128), torch.empty(1000, 128),
                                                 torch.zeros(300, dtype=torch.long)).shape_env
    assert not env.replacements and not env.guards
