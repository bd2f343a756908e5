"""How far a NaN in a key or value reaches in window_attention: rows that see it are NaN, rows more than 64 positions before it
or behind the last one that sees it have the bits they have without it, in outputs and in the queries' gradients.

The sizes fill the chip with blocks of four row tiles, whose 128 rows stage one set of keys: keys in the last tile of the first
keys that are none of them are there for the block's early rows and not for its late ones."""

import math

import pytest
import torch

from test_gpu_window import DEV, make, visible

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from tattn import hip_available

    assert hip_available(DEV), "libtattn_hip.so did not load or the device is not a gfx950"


CASES = [
    # z, h, hk, n, s, d, window, sinks, key, dtype
    (1, 24, 24, 1400, 1400, 128, 1024, 4, 4, torch.bfloat16),
    (1, 24, 24, 1400, 1400, 128, 500, 1, 13, torch.float16),
    (1, 28, 28, 1300, 1300, 64, 1024, 4, 31, torch.float16),
    (1, 28, 28, 1300, 1300, 64, 724, 40, 45, torch.bfloat16),
    (1, 45, 45, 1300, 1300, 32, 600, 70, 95, torch.bfloat16),   # first keys end two tiles behind where windows begin
    (2, 24, 24, 1300, 1300, 16, 90, 33, 40, torch.float16),
    (2, 24, 8, 900, 900, 64, 300, 4, 9, torch.float16),         # three heads' rows to a position
    (1, 24, 24, 1000, 1400, 128, 650, 4, 20, torch.bfloat16),   # the last queries of longer keys
    (1, 24, 24, 1400, 1400, 128, 512, 32, 33, torch.bfloat16),  # first keys end with a tile
    (1, 24, 24, 1400, 1400, 128, 512, 0, 700, torch.bfloat16),
    (1, 3, 3, 1400, 1400, 64, 1019, 4, 6, torch.float32),
    (1, 2, 2, 700, 700, 128, 305, 70, 80, torch.float32),
    (1, 2, 2, 1400, 1400, 64, 1019, 4, 6, torch.float16),       # few rows: one row tile per workgroup
]


@pytest.mark.parametrize("z,h,hk,n,s,d,window,sinks,key,dtype", CASES)
@pytest.mark.parametrize("where", ["k", "v"])
def test_a_nan_reaches_no_further_than_documented(z, h, hk, n, s, d, window, sinks, key, dtype, where):
    from tattn import window_attention

    print("reach", z, h, hk, n, s, d, window, sinks, key, dtype, where, flush=True)
    q, k, v, do = make(z, h, hk, n, s, d, dtype, seed=11)

    def run(k, v):
        leaf = q.clone().requires_grad_()
        o = window_attention(leaf, k, v, window, sinks)
        return o.detach(), torch.autograd.grad(o, leaf, do)[0]

    clean = run(k, v)
    bad = {"k": k.clone(), "v": v.clone()}
    bad[where][:, :, key] = math.nan
    got = run(bad["k"], bad["v"])
    sees = visible(1, n, s, window, sinks)[0, :, key]
    at = torch.arange(s - n, s, device=DEV)
    assert sinks <= key and sees.any()
    far = (at < key - 64) | (at > key + window - 1 + 64)
    assert far.any() and not (far & sees).any()
    for name, a, b in zip(("o", "dq"), got, clean):
        assert a[:, :, sees].isnan().all(), name
        hit = a[:, :, far].isnan().any(-1).any(0).any(0)
        assert not hit.any(), f"{name}: NaN in rows at {at[far][hit].tolist()}"
        assert torch.equal(a[:, :, far], b[:, :, far]), name
