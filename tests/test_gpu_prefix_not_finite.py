"""prefix_attention where an own value or key of a sequence's newest tokens is not finite: rows at positions before it are as if it
were not there, rows that see it are not finite in its column."""

import math

import pytest
import torch
from test_gpu_cross import BF16, DEV, F16, i32
from test_gpu_prefix import make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from tattn import hip_available

    assert hip_available(DEV), "libtattn_hip.so did not load or the device is not a gfx950"


@pytest.mark.parametrize("fill", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype,d", [(F16, 64), (BF16, 128), (F16, 32), (BF16, 16)])
@pytest.mark.parametrize("n,s,lens", [(2, 40, (40, 2)), (3, 40, (33, 7)), (5, 300, (300, 66)), (40, 200, (200, 41)), (70, 600, (600, 65))])
def test_own_values_reach_no_earlier_row(n, s, lens, dtype, d, fill):
    from tattn import prefix_attention

    q, pk, pv, k, v = make(1, 2, 4, 2, n, 50, s, d, dtype)
    ends, lens = lens, i32(*lens)
    for back in (1, 2, n // 2, n - 1):  # the key's place from the end
        at = [max(0, end - back) for end in ends]
        without, with_ = v.clone(), v.clone()
        for z, a in enumerate(at):
            without[z, :, a, 5] = 0.0
            with_[z, :, a, 5] = fill
        want = prefix_attention(q, pk, pv, k, without, lens)
        got = prefix_attention(q, pk, pv, k, with_, lens)
        for z, (a, end) in enumerate(zip(at, ends)):
            first = n - (end - a)  # the row that sits on the key
            print(n, s, d, dtype, "key", a, "first row", first, flush=True)
            assert torch.equal(got[z, :, :first], want[z, :, :first])
            assert not torch.isfinite(got[z, :, first:, 5]).any()
            others = [i for i in range(d) if i != 5]
            assert torch.equal(got[z][..., others], want[z][..., others])
