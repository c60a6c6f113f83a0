"""Sizes that the 4-bit serving operators refuse on the host, before anything is launched."""

from __future__ import annotations

import pytest

from mamba3_amd import _native

FAKE = 1 << 12  # an address that is never dereferenced: the call is refused first


@pytest.fixture(scope="module")
def lib():
    if not _native.LIB_PATH.exists():
        from mamba3_amd import build
        build.build(verbose=False)
    return _native.lib()


@pytest.mark.parametrize("rows,n", [(1 << 11, 1 << 25), (1 << 10, 1 << 26), (1 << 26, 1 << 26)])
def test_results_of_more_pieces_than_a_grid_has_room_for(lib, rows, n):
    assert lib.m3_mx_linear(rows, n, 64, 1, 1, FAKE, FAKE, FAKE, FAKE, None, 1.0, FAKE, None) == 3
