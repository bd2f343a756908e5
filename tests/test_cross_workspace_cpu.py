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


# A launch holds fewer than 2^32 threads; workgroups have 64 to 512. Refused before anything is launched, by the call that asks for the
# workspace and by the operator itself.
FWD, BWD = 0, 1
F16, F32 = 0, 1


def cross_workspace(*args):
    out = ctypes.c_int64()
    rc = _lib.load().tattn_cross_workspace(*args, ctypes.byref(out))
    return rc, _lib.last_error() if rc else out.value


@pytest.mark.parametrize("backward,z,n,s,d,dtype", [
    (FWD, 1 << 25, 1, 1, 16, F16),            # few keys, 256 threads
    (FWD, 1 << 24, 1, 200, 64, F16),          # few rows, 256
    (FWD, 1 << 18, 64 * 128, 200, 128, F16),  # many rows, 256
    (FWD, 1 << 24, 65, 200, 64, F32),
    (BWD, 1 << 25, 1, 1, 16, F16),
    (BWD, 1 << 23, 1, 200, 128, F16),         # dQ by pairs of waves, 512
    (BWD, 1 << 24, 1, 200, 64, F16),
    (BWD, 1 << 25, 1, 1, 16, F32),            # dK / dV
])
def test_launches_that_are_too_large_are_refused(backward, z, n, s, d, dtype):
    rc, text = cross_workspace(backward, z, 1, 1, n, s, d, dtype)
    assert rc == 1 and "grid too large" in text
    strides = (ctypes.c_int64 * 4)(n * d, n * d, d, 1)
    keys = (ctypes.c_int64 * 4)(s * d, s * d, d, 1)
    sizes = z, 1, 1, n, s, d, dtype, 1.0, None
    if backward:
        q, k = [strides], [keys]
        rc = _lib.load().tattn_cross_bwd(*[16] * 8, 16, None, 16, *q, *k, *k, *q, *q, *q, *k, *k, *sizes)
    else:
        rc = _lib.load().tattn_cross_fwd(16, 16, 16, 16, None, None, 16, strides, keys, keys, strides, *sizes)
    assert rc == 1 and "grid too large" in _lib.last_error()


@pytest.mark.parametrize("backward,z,n,s,d,dtype", [
    (FWD, (1 << 24) - 8, 1, 1, 16, F16), (BWD, (1 << 23) - 8, 1, 200, 128, F16), (FWD, 1 << 25, 1, 1, 16, F32), (BWD, (1 << 24) - 8, 1, 1, 16, F32),
])
def test_the_largest_launches_are_not(backward, z, n, s, d, dtype):
    assert cross_workspace(backward, z, 1, 1, n, s, d, dtype)[0] == 0


@pytest.mark.parametrize("groups,members,n,p,s", [(1 << 24, 1, 1, 1, 1), (1, 1 << 24, 1, 40, 40), (1 << 13, 1 << 11, 1, 1, 0), (1 << 10, 1 << 10, 130, 1, 1)])
def test_launches_behind_a_prefix_that_are_too_large_are_refused(groups, members, n, p, s):
    """The last: 136 million rows of 128 columns to be joined, eight a workgroup."""
    out = ctypes.c_int64()
    assert _lib.load().tattn_prefix_workspace(groups, members, 1, 1, n, p, s, 128, ctypes.byref(out)) == 1
    assert "grid too large" in _lib.last_error()
    a, b, c = ((ctypes.c_int64 * 4)(128 * x, 128 * x, 128, 1) for x in (n, p, s))
    rc = _lib.load().tattn_prefix_attention(*[16] * 6, None, 16, 16, a, b, b, c, c, a, groups, members, 1, 1, n, p, s, 128, 0, 1.0, None)
    assert rc == 1 and "grid too large" in _lib.last_error()
