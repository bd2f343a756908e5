"""What is not finite in a query or in a gradient's row, next to lengths shorter than the keys: keys at or past them get gradients
of zero, in the kernels for few keys as in the others."""

import math

import pytest
import torch
from test_gpu_cross import BF16, DEV, F16, F32, i32, make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from tattn import hip_available

    assert hip_available(DEV), "libtattn_hip.so did not load or the device is not a gfx950"


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("where", ["query", "gradient"])
@pytest.mark.parametrize("n,s,d,dtype", [
    (40, 60, 64, F16), (40, 60, 64, BF16), (40, 100, 64, F16), (40, 100, 64, BF16), (40, 20, 64, F16),
    (700, 60, 64, F16), (700, 100, 64, BF16), (700, 128, 64, F16),  # rows in parts
    (40, 60, 128, F16), (700, 30, 128, BF16), (700, 120, 32, F16), (40, 120, 16, BF16), (40, 50, 32, BF16),
    (40, 100, 128, F16), (40, 300, 64, F16), (700, 300, 64, BF16), (40, 100, 64, F32),
])
def test_keys_behind_the_lengths_get_zeros(n, s, d, dtype, where, value):
    from tattn import cross_attention

    q, k, v, do = make(3, 4, 2, n, s, d, dtype)
    lens = i32(s - 9, 1, 0)
    (q if where == "query" else do)[:, :, n // 2, 3] = value
    leaves = [t.requires_grad_() for t in (q, k, v)]
    _, dk, dv = torch.autograd.grad(cross_attention(*leaves, lens), leaves, do)
    behind = (torch.arange(s, device=DEV) >= lens[:, None])[:, None, :, None]
    for t in (dk, dv):
        assert not t.masked_select(behind).any()
        assert not torch.isfinite(t[0, :, : s - 9]).all()
