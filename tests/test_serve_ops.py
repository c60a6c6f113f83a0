"""Refusals of the operators that serve from 4-bit weights, on the host: nothing here launches a kernel."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import mamba3_amd
from mamba3_amd import MXTensor, _native

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


def test_quantize_refuses_bad_arguments(lib):
    def go(rows=4, k=64, dtype=1, gated=0, fmt=1, x=FAKE, data=FAKE, scales=FAKE):
        return lib.m3_mx_quantize(rows, k, dtype, gated, fmt, x, data, scales, None)

    assert go(x=None) == go(data=None) == go(scales=None) == 1
    assert go(rows=0) == go(k=0) == go(k=-3) == 2
    assert go(rows=(1 << 32) + 1) == go(k=(1 << 24) + 1) == go(dtype=2) == go(fmt=2) == go(fmt=-1) == 3
    assert go(x=FAKE + 1) == go(data=FAKE + 8) == go(scales=FAKE + 2) == go(x=FAKE + 2, dtype=0) == 5


def test_dequantize_refuses_bad_arguments(lib):
    def go(rows=4, k=64, fmt=1, dtype=1, data=FAKE, scales=FAKE, out=FAKE):
        return lib.m3_mx_dequantize(rows, k, fmt, dtype, data, scales, out, None)

    assert go(data=None) == go(scales=None) == go(out=None) == 1
    assert go(rows=0) == go(k=0) == 2
    assert go(k=(1 << 24) + 1) == go(dtype=7) == go(fmt=2) == 3
    assert go(data=FAKE + 4) == go(scales=FAKE + 1) == go(out=FAKE + 1) == 5


def test_add_rmsnorm_refuses_bad_arguments(lib):
    def fwd(rows=4, d=64, dtype=1, x=FAKE, res=FAKE, w=FAKE, total=FAKE, y=FAKE):
        return lib.m3_add_rmsnorm_fwd(rows, d, dtype, x, res, w, 1.0, 1e-5, total, y, None, None)

    for name in ("x", "res", "w", "total", "y"):
        assert fwd(**{name: None}) == 1 and fwd(**{name: FAKE + 1}) == 5
    assert fwd(rows=0) == fwd(d=0) == 2
    assert fwd(dtype=2) == fwd(d=(1 << 24) + 1) == fwd(rows=1 << 33) == 3

    def mx(rows=4, d=64, dtype=1, x=FAKE, res=FAKE, w=FAKE, total=FAKE, fmt=1, data=FAKE, scales=FAKE):
        return lib.m3_add_rmsnorm_mx(rows, d, dtype, x, res, w, 1.0, 1e-5, total, fmt, data, scales, None)

    for name in ("x", "res", "w", "total", "data", "scales"):
        assert mx(**{name: None}) == 1
    assert mx(fmt=3) == mx(dtype=-1) == 3 and mx(data=FAKE + 8) == mx(scales=FAKE + 1) == mx(total=FAKE + 1) == 5

    def bwd(rows=4, d=64, dtype=1, total=FAKE, w=FAKE, rstd=FAKE, dt=FAKE, dy=FAKE, dx=FAKE, dr=FAKE, dw=FAKE, ws=FAKE, n=1 << 40):
        return lib.m3_add_rmsnorm_bwd(rows, d, dtype, total, w, rstd, dt, dy, 1.0, dx, dr, dw, ws, n, None)

    for name in ("total", "w", "rstd", "dy"):
        assert bwd(**{name: None}) == 1
    assert bwd(rows=-1) == 2 and bwd(dtype=5) == 3 and bwd(dx=FAKE + 1) == 5 and bwd(ws=FAKE + 128) == 5
    assert bwd(ws=None) == bwd(n=4 * 64 - 1) == 4
    assert bwd(dx=None, dr=None, dw=None) == 0  # nothing to do


@pytest.mark.parametrize("rows,d", [(1, 1), (8192, 768), (3, 8193), (1 << 20, 20000)])
def test_add_rmsnorm_workspace(lib, rows, d):
    st, n = _size(lib.m3_add_rmsnorm_bwd_workspace_size, rows, d)
    assert st == 0 and 4 * d <= n <= 512 * 4 * d


def test_mx_linear_refuses_bad_arguments(lib):
    def go(rows=4, n=64, k=64, fmt=1, out_dtype=1, x=FAKE, xs=FAKE, w=FAKE, ws=FAKE, res=None, out=FAKE):
        return lib.m3_mx_linear(rows, n, k, fmt, out_dtype, x, xs, w, ws, res, 1.0, out, None)

    for name in ("x", "xs", "w", "ws", "out"):
        assert go(**{name: None}) == 1
    assert go(rows=0) == go(n=0) == go(k=0) == 2
    assert go(rows=(1 << 26) + 1) == go(n=(1 << 26) + 1) == go(k=(1 << 20) + 1) == go(fmt=2) == go(out_dtype=2) == 3
    assert go(x=FAKE + 8) == go(w=FAKE + 8) == go(xs=FAKE + 2) == go(ws=FAKE + 1) == go(out=FAKE + 1) == go(res=FAKE + 1) == 5


def test_sample_refuses_bad_arguments(lib):
    def go(rows=4, vocab=64, dtype=1, z=FAKE, u=FAKE, token=FAKE):
        return lib.m3_sample_tokens(rows, vocab, dtype, z, u, None, 1.0, None, 0, None, 1.0, None, 0.0, token, None, None)

    assert go(z=None) == go(u=None) == go(token=None) == 1
    assert go(rows=0) == go(vocab=0) == 2 and go(vocab=(1 << 22) + 1) == go(rows=(1 << 30) + 1) == go(dtype=2) == 3
    assert go(z=FAKE + 1) == 5


def test_python_refuses_cpu_tensors_and_bad_shapes():
    x = torch.randn(4, 64)
    w = MXTensor(torch.zeros(8, 64, dtype=torch.uint8), torch.zeros(8, 4, dtype=torch.uint8), (8, 64), "e2m1")
    for call in (lambda: mamba3_amd.quantize_mx(x), lambda: mamba3_amd.silu_mul_mx(x), lambda: w.dequantize(),
                 lambda: mamba3_amd.add_rms_norm(x, x, x[0]), lambda: mamba3_amd.add_rms_norm_mx(x, None, x[0]),
                 lambda: mamba3_amd.mx_linear(x, w), lambda: mamba3_amd.sample_tokens(x, torch.rand(4))):
        with pytest.raises(RuntimeError, match="GPU"):
            call()
    for call in (lambda: mamba3_amd.quantize_mx(x, "e5m2"), lambda: mamba3_amd.quantize_mx(torch.randn(3, 0)), lambda: mamba3_amd.quantize_mx(torch.tensor(1.0)),
                 lambda: mamba3_amd.silu_mul_mx(x[:, :63]), lambda: mamba3_amd.add_rms_norm(x, x[:3], x[0]),
                 lambda: mamba3_amd.add_rms_norm(x, x, x[0, :63]), lambda: mamba3_amd.add_rms_norm_mx(x, x.T, x[0]),
                 lambda: mamba3_amd.mx_linear(x, x), lambda: mamba3_amd.mx_linear(w, MXTensor(torch.zeros(8, 128, dtype=torch.uint8), w.scales, (8, 64), "e4m3")),
                 lambda: mamba3_amd.mx_linear(w, MXTensor(w.data, w.scales, (8, 65), "e2m1")),
                 lambda: mamba3_amd.mx_linear(w, w, torch.zeros(8, 7)), lambda: mamba3_amd.mx_linear(w, w, torch.zeros(8, 8), out_dtype=torch.bfloat16)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: mamba3_amd.quantize_mx(x.half()), lambda: mamba3_amd.quantize_mx(x.long()), lambda: w.dequantize(torch.float16),
                 lambda: mamba3_amd.add_rms_norm(x, x.bfloat16(), x[0]), lambda: mamba3_amd.add_rms_norm(x.double(), x.double(), x[0].double()),
                 lambda: mamba3_amd.mx_linear(w, w, out_dtype=torch.float16), lambda: mamba3_amd.sample_tokens(x.half(), torch.rand(4)),
                 lambda: mamba3_amd.sample_tokens(x, torch.rand(4).double()), lambda: mamba3_amd.sample_tokens(x, torch.rand(4), torch.rand(4).double()),
                 lambda: mamba3_amd.sample_tokens(x, torch.rand(4), top_k=torch.rand(4))):
        with pytest.raises(TypeError):
            call()


def test_python_refuses_gradients_where_there_is_no_backward():
    x = torch.randn(4, 64, requires_grad=True)
    w = MXTensor(torch.zeros(8, 64, dtype=torch.uint8), torch.zeros(8, 4, dtype=torch.uint8), (8, 64), "e2m1")
    for call in (lambda: mamba3_amd.quantize_mx(x), lambda: mamba3_amd.silu_mul_mx(x), lambda: mamba3_amd.add_rms_norm_mx(x, x, x[0]),
                 lambda: mamba3_amd.mx_linear(x, w), lambda: mamba3_amd.mx_linear(w, w, torch.zeros(8, 8, requires_grad=True)),
                 lambda: mamba3_amd.sample_tokens(x, torch.rand(4), return_logprob=True)):
        with pytest.raises(RuntimeError, match="no backward"):
            call()


@pytest.mark.parametrize("bad", [dict(temperature=-1.0), dict(temperature=math.nan), dict(top_k=-1), dict(top_p=1.5), dict(top_p=-0.1), dict(min_p=2.0),
                                 dict(min_p=math.nan), dict(temperature=torch.rand(3)), dict(top_p=torch.rand(4, 1))])
def test_sample_refuses_bad_settings(bad):
    with pytest.raises(ValueError):
        mamba3_amd.sample_tokens(torch.randn(4, 10), torch.rand(4), **bad)


def test_sample_refuses_bad_shapes():
    for z, u in ((torch.randn(4, 10), torch.rand(5)), (torch.tensor(1.0), torch.rand(())), (torch.randn(4, 0), torch.rand(4)),
                 (torch.empty(1, (1 << 22) + 1, dtype=torch.bfloat16), torch.rand(1))):
        with pytest.raises(ValueError):
            mamba3_amd.sample_tokens(z, u)


def test_mxtensor_refuses_what_does_not_fit():
    data, scales = torch.zeros(6, 128, dtype=torch.uint8), torch.zeros(6, 4, dtype=torch.uint8)
    t = MXTensor(data, scales, (2, 3, 100), "e4m3")
    assert t.shape == (2, 3, 100) and t.device.type == "cpu" and "e4m3" in repr(t)
    for args in ((data, scales, (2, 3, 129), "e4m3"), (data, scales, (6, 100), "e2m1"), (data, scales, (5, 100), "e4m3"), (data, scales, (), "e4m3"),
                 (data, scales, (6, 0), "e4m3"), (data.int(), scales, (6, 100), "e4m3"), (data, scales[:, :3], (6, 100), "e4m3"),
                 (data.t().contiguous().t(), scales, (6, 100), "e4m3"), (data, scales, (6, 100), "int8")):
        with pytest.raises(ValueError):
            MXTensor(*args)


def test_header_names_the_stored_layout():
    assert [_native.mx_padded(k) for k in (1, 128, 129, 500)] == [128, 128, 256, 512]
    assert _native.mx_row_bytes(500, "e4m3") == 512 and _native.mx_row_bytes(500, "e2m1") == 256


def test_python_refuses_what_does_not_go_in_front_of_a_product():
    x = torch.randn(4, 64)
    w = MXTensor(torch.zeros(8, 64, dtype=torch.uint8), torch.zeros(8, 4, dtype=torch.uint8), (8, 64), "e2m1")
    for call in (lambda: mamba3_amd.mx_linear(w, w, gated=True), lambda: mamba3_amd.mx_linear(w, w, norm_weight=x[0]), lambda: mamba3_amd.mx_linear(x, w, gated=True),
                 lambda: mamba3_amd.mx_linear(torch.randn(4, 128), w, norm_weight=x[0], gated=True), lambda: mamba3_amd.mx_linear(x, w, norm_weight=x[0, :63]),
                 lambda: mamba3_amd.mx_linear(x, w, norm_weight=x), lambda: mamba3_amd.mx_linear(x, w, norm_weight=x[0].bfloat16())):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError, match="no backward"):
        mamba3_amd.mx_linear(x, w, norm_weight=x[0].clone().requires_grad_())


def test_mx_linear_tensor_refuses_bad_arguments(lib):
    def go(rows=4, n=8, k=64, x_dtype=0, out_dtype=0, before=0, x=FAKE, norm=None, w=FAKE, ws=FAKE, res=None, out=FAKE):
        return lib.m3_mx_linear_tensor(rows, n, k, x_dtype, out_dtype, before, x, norm, 1e-5, w, ws, res, 1.0, out, None)

    assert go(x=None) == go(w=None) == go(ws=None) == go(out=None) == go(before=1) == 1
    assert go(rows=0) == go(n=0) == go(k=0) == 2
    assert go(before=3) == go(before=-1) == go(x_dtype=2) == go(out_dtype=2) == go(rows=17) == go(k=6145) == go(n=(1 << 26) + 1) == 3
    assert go(before=1, norm=FAKE, k=2049) == go(before=1, norm=FAKE, out_dtype=1) == go(before=2, out_dtype=1) == 3
    assert go(x=FAKE + 2) == go(w=FAKE + 8) == go(ws=FAKE + 2) == go(out=FAKE + 2) == go(res=FAKE + 1) == go(before=1, norm=FAKE + 1) == 5


def test_model_refuses_what_it_cannot_serve():
    lm = mamba3_amd.KulaMambaLM(50, 64, n_layers=1, d_state=16, headdim=16, mimo_rank=1)
    with pytest.raises(RuntimeError, match="GPU"):
        lm.quantize_mx()
    assert not lm.mx_weights and not lm.layers[0].mx_weights
    biased = mamba3_amd.KulaMambaLM(50, 64, n_layers=1, d_state=16, headdim=16, mimo_rank=1, bias=True)
    with pytest.raises(RuntimeError, match="bias"):
        biased.quantize_mx()
    ids = torch.zeros(1, 3, dtype=torch.long)
    for bad in (dict(top_p=1.5), dict(min_p=-0.1), dict(top_p=0.5, top_k=0), dict(top_p=0.5, temperature=-1.0), dict(min_p=math.nan)):
        with pytest.raises(ValueError, match="top_p"):
            lm.generate(ids, 1, **bad)


def test_mx_linear_exact_refuses_bad_arguments(lib):
    import ctypes
    size = ctypes.c_size_t(0)
    assert lib.m3_mx_linear_exact_workspace_size(1024, 10000, 1024, ctypes.byref(size)) == 0 and size.value == (1024 + 10000) * 1024 * 2
    assert lib.m3_mx_linear_exact_workspace_size(255, 1 << 20, 1024, ctypes.byref(size)) == 0 and size.value == 0
    assert lib.m3_mx_linear_exact_workspace_size(0, 1024, 1024, ctypes.byref(size)) == 2 and lib.m3_mx_linear_exact_workspace_size(1024, 1024, 1024, None) == 1

    def go(rows=1024, n=10000, k=1024, fmt=1, x=FAKE, xs=FAKE, w=FAKE, ws=FAKE, res=None, out=FAKE, room=FAKE, bytes_=1 << 30):
        return lib.m3_mx_linear_exact(rows, n, k, fmt, x, xs, w, ws, res, 1.0, out, room, bytes_, None)

    assert go(x=None) == go(xs=None) == go(w=None) == go(ws=None) == go(out=None) == 1
    assert go(rows=0) == go(n=-1) == go(k=0) == 2
    assert go(rows=16) == go(n=8) == go(fmt=2) == go(k=(1 << 20) + 1) == 3
    assert go(x=FAKE + 8) == go(w=FAKE + 8) == go(xs=FAKE + 2) == go(ws=FAKE + 1) == go(out=FAKE + 2) == go(res=FAKE + 2) == 5
    assert go(room=None) != 0 and go(bytes_=100) != 0
