"""Workspaces of attention over another length and behind a prefix: regions that start on 16 bytes."""

import ctypes

import pytest

from tattn import _lib


def prefix_floats(*sizes):
    out = ctypes.c_int64()
    assert _lib.load().tattn_prefix_workspace(*sizes, ctypes.byref(out)) == 0, _lib.last_error()
    return out.value


@pytest.mark.parametrize("d", [16, 32, 64, 128])
@pytest.mark.parametrize("rows", [1, 3, 5])
def test_own_parts_start_on_16_bytes(rows, d):
    """One part of the prefix and one of the own keys: a region of rows (dim + 2) floats each, the second behind the first on a multiple
    of four floats."""
    region = rows * (d + 2)
    assert prefix_floats(1, 1, rows, 1, 1, 1, 1, d) >= (region + 3) // 4 * 4 + region
