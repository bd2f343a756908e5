"""cache4_attention where each wave takes many key tiles: many requests over long tables, whole and in parts, against float64
over the held values. Bounds as in test_gpu_cache4_attention.py.

How many tiles a workgroup takes is the library's rule, seen here through the size of the workspace."""

import ctypes

import pytest
import torch

from tattn import _lib
from test_gpu_cache4_attention import DEV, check, make

CASES = [
    # requests, longest, h, hk, d, page, window, sinks, dtype
    (64, 2000, 16, 8, 128, 16, 0, 0, torch.bfloat16),
    (25, 6000, 8, 4, 128, 16, 0, 0, torch.float16),
    (30, 5000, 40, 1, 128, 32, 0, 0, torch.bfloat16),     # three groups of heads to a key head
    (128, 1500, 4, 4, 64, 16, 0, 0, torch.float16),
    (24, 6000, 12, 4, 64, 16, 0, 0, torch.bfloat16),
    (64, 4000, 8, 4, 64, 16, 1500, 40, torch.float16),
    (40, 5000, 6, 3, 32, 32, 0, 0, torch.bfloat16),
    (90, 1500, 6, 6, 32, 16, 0, 0, torch.float16),
    (60, 5000, 4, 2, 128, 64, 3000, 4, torch.bfloat16),
]


def tiles_and_parts(r, longest, h, hk, d, page, window, sinks):
    """Key tiles of the longest request, and the parts they are cut into."""
    width = (longest + page - 1) // page
    out = ctypes.c_int64()
    assert _lib.load().tattn_cache4_attention_workspace(r, h, hk, d, width, page, window, sinks, ctypes.byref(out)) == 0
    seen = min(width * page, window + sinks) if window else width * page
    return seen // 32, max(1, out.value // (r * h * (d + 2)))


@pytest.mark.parametrize("case", CASES)
def test_each_of_four_waves_takes_at_least_three_tiles(case):
    tiles, parts = tiles_and_parts(*case[:8])
    assert tiles / parts >= 12


def test_both_whole_and_in_parts():
    for d in (32, 64, 128):
        assert {tiles_and_parts(*c[:8])[1] > 1 for c in CASES if c[4] == d} == {True, False}


@pytest.fixture(scope="module")
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from tattn import hip_available

    assert hip_available(DEV), "libtattn_hip.so did not load or the device is not a gfx950"


@pytest.mark.gpu
@pytest.mark.parametrize("r,longest,h,hk,d,page,window,sinks,dtype", CASES)
def test_matches_float64_over_the_held_values(gpu, r, longest, h, hk, d, page, window, sinks, dtype):
    from tattn import cache4_attention

    print("long tables", r, longest, h, hk, d, page, window, sinks, dtype, flush=True)
    q, cache, tables, lens = make(r, longest, h, hk, d, page, dtype, seed=31)
    lens[6:9] = longest  # whole tables besides the random lengths
    got = cache4_attention(q, cache, tables, lens, window=window or None, sinks=sinks)
    check("o", got, q, cache, tables, lens, window, sinks, d ** -0.5)
    assert torch.equal(got, cache4_attention(q, cache, tables, lens, window=window or None, sinks=sinks))
    garbage = torch.tensor([-1, cache.pages, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=DEV)
    tables[:, 2::5] = garbage[torch.arange(tables[:, 2::5].shape[1], device=DEV) % 4]
    got = cache4_attention(q, cache, tables, lens, window=window or None, sinks=sinks)
    check("holes", got, q, cache, tables, lens, window, sinks, d ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("r,longest,h,hk,d,page,window,sinks,dtype", CASES)
@pytest.mark.parametrize("falling", [False, True])
def test_scores_that_grow_or_fall_along_the_sequence(gpu, r, longest, h, hk, d, page, window, sinks, dtype, falling):
    """K's exponents go from 2^-9 to 2^3 along every request: the largest score is passed again and again until the last tiles,
    or lies in the first ones."""
    from tattn import cache4_attention

    print("growing", r, longest, h, hk, d, page, window, sinks, dtype, falling, flush=True)
    q, cache, tables, lens = make(r, longest, h, hk, d, page, dtype, seed=32)
    lens[6:9] = longest
    at = torch.arange(tables.shape[1] * page, device=DEV)
    e = 118 + 12 * at // at.numel()
    e = (e.flip(0) if falling else e).to(torch.uint8).view(-1, page)  # [width, page]
    cache.scales[tables.long(), :, 0] = e[None, :, None, :, None]
    got = cache4_attention(q, cache, tables, lens, window=window or None, sinks=sinks)
    check("o", got, q, cache, tables, lens, window, sinks, d ** -0.5)
