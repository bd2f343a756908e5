"""Gradients of cross_attention in float16 where dS passes the type's largest value and the results do not: on both sides of where the
kernels for few keys end (128 keys, 64 at head dim 128), with rows and keys in parts, and with small rows beside the large.

Bounds of test_gpu_cross. dS is then held in steps of up to f' = 2^-25 2^b, b the power of two that it is divided by, which keeps
|dO| |v| 2^1 (|dS| = P |dP - delta|, each term at most |dO| |v|) below 2^16 and is taken from norms known to a factor of two each, or, where
the keys' norms are not known beforehand, from the largest that values of the type have, 65,504 sqrt(D) < 2^20: b <= e + 7 with 2^e <= |dO|. So
f' <= 2^-25 max(2^7 |dO|, 2^-11 |dO| |v|) of the largest rows. For dK it is V that is divided, in its own type: dP is then off by up to
sqrt(D) 2^-25 2^b |dO|, here b <= log2(|dO| |v|) - 11 of the largest."""

import pytest
import torch
from test_gpu_cross import DEV, F16, close, i32, make, plain, visible

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from tattn import hip_available

    assert hip_available(DEV), "libtattn_hip.so did not load or the device is not a gfx950"


def check(q, k, v, do, lens, scale):
    from tattn import cross_attention

    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = cross_attention(*leaves, lens, sm_scale=scale)
    grads = torch.autograd.grad(o, leaves, do)
    z, h, n, d = q.shape
    g = h // k.shape[1]
    see = visible(z, n, k.shape[2], lens)
    want = plain(q, k, v, do, see, scale)
    rows, keys = do.double().norm(dim=-1, keepdim=True), v.double().norm(dim=-1).max()
    most = rows.amax((1, 2), keepdim=True)  # of a sequence
    step = 2.0 ** -25 * torch.maximum(2.0 ** 7 * rows, 2.0 ** -11 * rows * keys)
    step_all = 2.0 ** -25 * torch.maximum(2.0 ** 7 * most, 2.0 ** -11 * most * keys)
    kd, qd = k.double().repeat_interleave(g, 1), q.double()
    p = torch.softmax((qd @ kd.transpose(2, 3).contiguous() * scale).masked_fill(~see[:, None], -torch.inf), -1)
    steps = step_all + p * d ** 0.5 * 2.0 ** -36 * most * keys * rows
    more = {"dq": step * (see[:, None].double() @ kd.abs()) * abs(scale),
            "dk": (steps.transpose(2, 3).contiguous() @ qd.abs()).reshape(z, -1, g, k.shape[2], d).sum(2) * abs(scale), "dv": 0.0}
    ds = (do.double() @ v.double().repeat_interleave(g, 1).transpose(2, 3).contiguous()).abs().max().item()
    assert ds > 65504, "dP passes the type"
    for name, got in zip(("dq", "dk", "dv"), grads):
        assert torch.isfinite(want[name][0]).all() and want[name][0].abs().max() < 60000
        close(name, got, want[name][0], want[name][1] + more[name])


@pytest.mark.parametrize("n,s,d", [
    (64, 60, 64), (64, 128, 64), (64, 129, 64), (64, 600, 64), (200, 64, 128), (200, 65, 128), (200, 128, 128), (200, 700, 128),
    (64, 129, 32), (64, 500, 16), (2, 3000, 64), (2, 3000, 128), (500, 140, 64), (130, 64, 32),
])
def test_values_and_gradients_are_large(n, s, d):
    q, k, v, do = make(2, 4, 2, n, s, d, F16)
    check(q / 256, k / 1024, v * 2048, do * 4096, i32(s, s - 5), d ** -0.5)


@pytest.mark.parametrize("n,s,d", [(64, 128, 64), (64, 129, 64), (200, 64, 128), (200, 65, 128), (300, 700, 32)])
def test_two_keys_share_all(n, s, d):
    """The largest dS that there are: values of both signs at the type's limit."""
    q, k, v, do = make(1, 2, 1, n, s, d, F16)
    v, do = torch.full_like(v, 60000.0), torch.full_like(do, 2.0 ** 6)
    v[:, :, 1::2] *= -1
    do = do * torch.rand(do.shape[:3], generator=torch.Generator().manual_seed(s)).to(DEV, F16)[..., None]
    check(q / 256, k / 2048, v, do, i32(2), d ** -0.5 / 64)


@pytest.mark.parametrize("s,d", [(60, 128), (65, 128), (100, 64), (128, 64), (129, 64), (50, 32), (200, 32), (120, 16)])
def test_rows_and_values_at_the_limit_of_the_type(s, d):
    """dS of 2^36 at a scale of 2^-30."""
    q, k, v, do = make(1, 2, 2, 2, s, d, F16)
    v, do = torch.full_like(v, 60000.0), torch.full_like(do, 30000.0)
    v[:, :, 1::2] *= -1
    check(q, k, v, do, i32(2), 2.0 ** -30)


@pytest.mark.parametrize("n,s,d", [(64, 128, 64), (64, 129, 64), (200, 65, 128), (300, 700, 32)])
def test_small_rows_beside_large_ones(n, s, d):
    """Every row of dQ is held to a bound of its own."""
    q, k, v, do = make(2, 4, 2, n, s, d, F16)
    do = do * 4096
    do[:, :, ::2] *= 2.0 ** -20
    check(q / 256, k / 1024, v * 2048, do, None, d ** -0.5)
