"""Limits of the quantisation entry points, refused on the host."""

from __future__ import annotations

import ctypes

import pytest

from kernels import _native


@pytest.mark.parametrize("rows,cols", [(1 << 31, 8), (1 << 30, 256), ((1 << 62) + 1, 512), (1 << 55, 1 << 20),
                                       ((1 << 63) - 1, 1), (1, (1 << 63) - 1), (2, 1 << 38)])
def test_quantisations_of_too_many_blocks_are_refused(rows, cols):
    """Blocks are counted in 32 bits; a count that wraps in 64 must not pass for a small one."""
    lib = _native.load()
    buf = ctypes.create_string_buffer(256)
    at = (ctypes.addressof(buf) + 127) // 128 * 128
    assert lib.quantize_rows_launch(at, rows, cols, cols, 1, at, cols, at, None) == _native.STATUS_INVALID
    # As many matrices of one block row each.
    assert lib.quantize_blocks_launch(at, rows, 1, cols, cols, cols, 1, at, at, None) == _native.STATUS_INVALID
