"""Pairs of qk_rope_axes without an axis stay as they are, whatever they hold: an infinity or a NaN in one of a pair does not reach
the other, and zeros keep their sign."""

import math

import pytest
import torch
from test_gpu_cross import BF16, DEV, F16, F32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from tattn import hip_available

    assert hip_available(DEV), "libtattn_hip.so did not load or the device is not a gfx950"


def same(a, b):
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) and torch.equal(a.signbit() & ~a.isnan(), b.signbit() & ~b.isnan())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("axes", ["quads", "single"])
@pytest.mark.parametrize("d", [16, 64, 128])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_unturned_pairs_stay_as_they_are(dtype, d, axes, interleaved):
    from tattn import qk_rope_axes

    half = d // 2
    axes = [(-1, 0)[i // 4 % 2] for i in range(half)] if axes == "quads" else [(-1, 0, -1)[i % 3] for i in range(half)]
    gen = torch.Generator().manual_seed(d)
    q, k, gq, gk = (torch.randn(2, h, 5, d, generator=gen).to(DEV, dtype) for h in (5, 2, 5, 2))
    cos, sin = (torch.rand(9, half, generator=gen).to(DEV) for _ in range(2))
    positions = torch.randint(0, 9, (1, 5), generator=gen).int().to(DEV)
    still = torch.tensor([a < 0 for a in axes], device=DEV)
    still = still.repeat_interleave(2) if interleaved else torch.cat((still, still))
    values = torch.tensor([math.inf, -math.inf, math.nan, -0.0, 0.0, -2.0], device=DEV, dtype=dtype)
    clean = qk_rope_axes(q, k, cos, sin, positions, axes, interleaved)
    for t in (q, k, gq, gk):
        t[..., still] = values[torch.randint(0, 6, t[..., still].shape, generator=gen).to(DEV)]
    leaves = [t.clone().requires_grad_() for t in (q, k)]
    out = qk_rope_axes(*leaves, cos, sin, positions, axes, interleaved)
    grads = torch.autograd.grad(out, leaves, (gq, gk))
    for got, x in zip((*out, *grads), (q, k, gq, gk)):
        assert same(got[..., still], x[..., still])
    for got, want in zip(out, clean):
        assert torch.equal(got[..., ~still], want[..., ~still])
    with torch.no_grad():
        nothing = qk_rope_axes(q, k, cos, sin, positions, (-1,) * half, interleaved)
    for got, x in zip(nothing, (q, k)):
        assert same(got, x)
