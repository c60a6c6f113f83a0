"""Tile and split choice of the tiled products (csrc/m3_gemm_plan.h), on the host: the header's search, compiled
with the host compiler, against every choice of its own estimate."""

from __future__ import annotations

import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest

from mamba3_amd import _native

ROOT = Path(__file__).resolve().parents[1]
SOURCE = r"""
#include "m3_gemm_plan.h"
using namespace m3;
// us of the chosen plan, of the best one of a single launch with any number of parts, the chosen parts
extern "C" void pair(int bf16, int64_t r0, int64_t c0, int64_t k0, int most0, int64_t r1, int64_t c1, int64_t k1, int most1,
                     double* us, int* parts) {
    const GemmTask t[2] = {{r0, c0, k0, most0, false}, {r1, c1, k1, most1, true}};
    const GemmPairPlan p = pair_plan(t, [&](const GemmTask (&v)[2]) { return search_plan(bf16, v, 2); });
    us[0] = p.apart ? p.p[0].us + p.p[1].us + 5.0 : p.p[0].us;
    parts[0] = p.p[0].splits[0], parts[1] = p.p[1].splits[1];
    us[1] = 1e30;
    for (int tile = bf16 ? kTileL : kTileM; tile <= kTileS; ++tile)
        for (int i = 1; i <= most0 && i <= k0; ++i)
            for (int j = 1; j <= most1 && j <= k1; ++j) {
                const int s[kGroupMax] = {i, j, 1, 1};
                us[1] = std::min(us[1], group_us(tile_costs(bf16)[tile], t, s, 2));
            }
}
"""


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(SOURCE)
    subprocess.run([cxx, "-O2", "-std=c++17", "-shared", "-fPIC", f"-I{ROOT / 'mamba3_amd' / 'csrc'}", f"-I{ROOT / 'include'}",
                    str(d / "plan.cpp"), "-o", str(d / "plan.so")], check=True)
    lib = ctypes.CDLL(str(d / "plan.so"))
    i64, i32 = ctypes.c_int64, ctypes.c_int
    lib.pair.argtypes = [i32, i64, i64, i64, i32, i64, i64, i64, i32, ctypes.POINTER(ctypes.c_double), ctypes.POINTER(i32)]
    lib.pair.restype = None
    return lib


def _piece(rows, vocab, size):
    """Columns of a piece of the vocabulary in the loss's backward."""
    most = min(max((256 << 20) // (rows * size) // 256 * 256, 256), 1 << 20)
    pieces = -(-vocab // most)
    if pieces == 1:
        return -(-vocab * size // 16) * 16 // size
    return -(-(-(-vocab // pieces)) // 256) * 256


@pytest.mark.parametrize("bf16", [True, False], ids=["bf16", "fp32"])
def test_loss_gradients_plan_is_near_the_best(plans, bf16):
    """dh (rows x d over the vocabulary) beside dW (vocabulary x d over the rows): no more than an eighth, or 2 us,
    above the best of all numbers of parts (the search tries every number to 8, then steps of an eighth to a third)."""
    size = 2 if bf16 else 4
    step = 128 // size
    us, parts = (ctypes.c_double * 2)(), (ctypes.c_int * 2)()
    for rows in (1, 3, 16, 60, 128, 300, 512, 777, 1024, 2048, 3000, 4096):
        for d in (64, 100, 256, 500, 768, 2048):
            for vocab in (200, 1000, 4099, 32000, 50021, 128000):
                piece = _piece(rows, vocab, size)
                plans.pair(bf16, rows, d, -(-piece // step), 64, piece, d, -(-rows // step), 16, us, parts)
                assert us[0] <= max(us[1] * 1.125, us[1] + 2.0), (rows, d, vocab, list(us), list(parts))


@pytest.mark.parametrize("dtype,rows,d,vocab,least", [
    (0, 16, 2048, 32000, 16), (0, 128, 2048, 128000, 16), (0, 512, 2048, 32000, 8), (0, 2048, 2048, 32000, 2),
    (1, 16, 2048, 50021, 16), (1, 1024, 2048, 50021, 4), (1, 512, 2048, 128000, 12), (0, 16, 64, 128000, 48),
    (0, 2048, 64, 2000, 4)])
def test_loss_of_few_rows_cuts_its_long_product(dtype, rows, d, vocab, least):
    """The library's own choice, seen in its workspace: the partial sums are what both gradients need more than
    none (dW, of many tiles, is not cut here)."""
    if not _native.LIB_PATH.exists():
        from mamba3_amd import build
        build.build(verbose=False)
    need = []
    for wanted in (0, 1):
        n = ctypes.c_size_t(0)
        assert _native.lib().m3_linear_xent_bwd_workspace_size(rows, d, vocab, dtype, wanted, wanted, ctypes.byref(n)) == 0
        need.append(n.value)
    parts = (need[1] - need[0]) // (rows * d * 4)
    assert parts >= least, (parts, need)
