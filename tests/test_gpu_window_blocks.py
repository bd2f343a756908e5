"""window_attention against float64 at sizes that fill the chip: the forward by blocks of four row tiles that every training
step and prompt runs, with its shorter blocks at the ends placed last. Bounds as in test_gpu_window.py.

Which kernel a size takes is the library's rule; that these sizes take this one is checked through it without a GPU."""

import math

import pytest
import torch

from tattn import _lib
from test_gpu_window import DEV, close, make, plain, visible

CASES = [
    # z, h, hk, n, s, d, window, sinks, dtype, layout
    (33, 1, 1, 513, 513, 128, 100, 4, torch.float16, "heads"),
    (11, 12, 4, 300, 300, 128, 90, 0, torch.bfloat16, "tokens"),
    (17, 8, 4, 130, 400, 128, 150, 5, torch.bfloat16, "heads"),   # the last queries of longer keys
    (2, 8, 8, 2500, 2500, 128, 700, 4, torch.float16, "tokens"),
    (60, 1, 1, 600, 600, 64, 200, 33, torch.bfloat16, "heads"),
    (20, 12, 4, 250, 250, 64, 70, 0, torch.float16, "tokens"),
    (30, 6, 3, 170, 500, 64, 300, 5, torch.float16, "heads"),
    (2, 8, 8, 2500, 2500, 64, 333, 70, torch.bfloat16, "tokens"),
    (101, 1, 1, 513, 513, 32, 64, 4, torch.float16, "heads"),
    (21, 20, 4, 150, 260, 32, 100, 40, torch.bfloat16, "tokens"),
    (90, 2, 2, 600, 600, 16, 128, 3, torch.bfloat16, "heads"),
    (50, 9, 3, 120, 120, 16, 1000, 0, torch.float16, "tokens"),
]

LENS = [
    # z, h, hk, n, s, d, window, sinks, dtype, layout
    (40, 8, 4, 200, 700, 128, 150, 4, torch.bfloat16, "tokens"),
    (45, 2, 2, 300, 500, 64, 100, 40, torch.float16, "heads"),
    (60, 6, 3, 150, 300, 32, 1000, 0, torch.bfloat16, "tokens"),
]


@pytest.mark.parametrize("case", CASES + LENS)
def test_these_sizes_take_blocks_of_four_row_tiles(case):
    z, h, hk, n, s, d, window, sinks = case[:8]
    assert _lib.load().tattn_window_picked(z, h, hk, n, s, d, window, sinks) == 0


def test_few_rows_share_their_keys():
    """The other side of the rule: one row tile per workgroup, its keys whole or in parts."""
    picked = _lib.load().tattn_window_picked
    assert picked(1, 8, 2, 257, 257, 128, 64, 4) >= 1
    assert picked(1, 8, 2, 1, 8192, 64, 8192, 0) > 1
    assert picked(1, 8, 3, 1, 8192, 64, 8192, 0) == -1 and "evenly" in _lib.last_error()


@pytest.fixture(scope="module")
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from tattn import hip_available

    assert hip_available(DEV), "libtattn_hip.so did not load or the device is not a gfx950"


@pytest.mark.gpu
@pytest.mark.parametrize("z,h,hk,n,s,d,window,sinks,dtype,layout", CASES)
def test_outputs_and_gradients_match_float64(gpu, z, h, hk, n, s, d, window, sinks, dtype, layout):
    from tattn import window_attention

    print("blocks", z, h, hk, n, s, d, window, sinks, dtype, layout, flush=True)
    q, k, v, do = make(z, h, hk, n, s, d, dtype, layout, seed=21)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o = window_attention(q, k, v, window, sinks)
    grads = torch.autograd.grad(o, leaves, do)
    with torch.no_grad():
        want = plain(q, k, v, do, window, sinks, d ** -0.5)
        for name, got in zip(("o", "dq", "dk", "dv"), (o, *grads)):
            close(name, got, *want[name])
        assert torch.equal(window_attention(q, k, v, window, sinks), o)
    o2 = window_attention(q, k, v, window, sinks)
    for a, b in zip(torch.autograd.grad(o2, leaves, do), grads):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("z,h,hk,n,s,d,window,sinks,dtype,layout", LENS)
def test_lengths_and_garbage_behind_them(gpu, z, h, hk, n, s, d, window, sinks, dtype, layout):
    from tattn import window_attention

    print("blocks, lens", z, h, hk, n, s, d, window, sinks, dtype, layout, flush=True)
    q, k, v, _ = make(z, h, hk, n, s, d, dtype, layout, seed=22)
    gen = torch.Generator().manual_seed(z + s)
    lens = torch.randint(1, s + 1, (z,), generator=gen, dtype=torch.int32)
    lens[:6] = torch.tensor([0, 1, n - 1, s, s + 100, -5])
    want = plain(q, k, v, None, window, sinks, d ** -0.5, lens)["o"]
    clean = window_attention(q, k, v, window, sinks, lens=lens.to(DEV))
    close("o", clean, *want)
    see = visible(z, n, s, window, sinks, lens)
    bad = torch.tensor([math.nan, math.inf, -math.inf], device=DEV, dtype=dtype)
    fill = bad[torch.arange(s, device=DEV) % 3][None, None, :, None]
    for t in (k, v):
        t.copy_(torch.where(see.any(1)[:, None, :, None], t, fill))
    assert torch.equal(window_attention(q, k, v, window, sinks, lens=lens.to(DEV)), clean)
    empty = ~see.any(-1)
    assert empty.any() and (clean.transpose(1, 2)[empty] == 0).all()
