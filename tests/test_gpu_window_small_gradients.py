"""window_attention in float16 with output gradients far below 1, as losses averaged over many tokens give them: dQ, dK and dV
keep the precision that they have for larger ones.

Bounds as in test_gpu_window.py but for the steps of 2^-24 below float16's normal range. dS, the operand of dQ and dK, is scaled
up by a power of two before it is rounded, 2^t with t = -floor(log2 of |dO|), |dO| the norm of a query's row (dQ) or the largest
among the rows that see a block of keys (dK), t between 0 and 15; so the absolute term of its rounding is
2^-25 2^-t <= 2^-25 max(min(|dO|, 1), 2^-15). Where the factor is in the exponent, t - M is rounded once more: a probability is
off by 64 2^-24 at most, relatively, for |t - M| below 64.
"""

import math

import pytest
import torch

from test_gpu_window import DEV, S32, close, make, visible

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from tattn import hip_available

    assert hip_available(DEV), "libtattn_hip.so did not load or the device is not a gfx950"


def bounds(q, k, v, do, window, sinks, scale):
    """{name: (value, bound)} of the gradients, in float64."""
    u = 2.0 ** -11
    z, h, n, d = q.shape
    hk, s = k.shape[1:3]
    g = h // hk
    see = visible(z, n, s, window, sinks)[:, None]
    qd, kd, vd, g64 = q.double(), k.double().repeat_interleave(g, 1), v.double().repeat_interleave(g, 1), do.double()
    kt, vt = kd.transpose(2, 3).contiguous(), vd.transpose(2, 3).contiguous()
    e = ((d + 4) * S32 * (qd.abs() @ kt.abs()) * abs(scale)).masked_fill(~see, 0.0).amax(-1, keepdim=True) + 2.0 ** -20 + 64 * S32
    p = torch.softmax(((qd @ kt) * scale).masked_fill(~see, -math.inf), -1)
    o = p @ vd
    eo = (p @ vd.abs()) * (2 * u + 2 * e + s * S32) + 2.0 ** -25 * (see.double() @ vd.abs()) + u * o.abs()
    dp, delta = g64 @ vt, (g64 * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    edp = (d + 4) * S32 * (g64.abs() @ vt.abs())
    edelta = (g64.abs() * (eo + (d + 4) * S32 * o.abs())).sum(-1, keepdim=True)
    ep = p * (2 * u + 2 * e)
    norm = g64.norm(dim=-1, keepdim=True)
    row, top = (2.0 ** -25 * x.clamp(2.0 ** -15, 1.0) for x in (norm, norm.amax()))
    eds = ep * (dp - delta).abs() + p * (edp + edelta)

    def t(x):
        return x.transpose(2, 3).contiguous()

    def group(x):
        return x.reshape(z, hk, g, s, d).sum(2)

    dq, edq = ds @ kd * scale, (eds + row * see + s * S32 * ds.abs()) @ kd.abs() * abs(scale)
    dk, edk = group(t(ds) @ qd) * scale, group(t(eds + top * see + n * g * S32 * ds.abs()) @ qd.abs()) * abs(scale)
    dv, edv = group(t(p) @ g64), group(t(ep + 2.0 ** -25 * see + n * g * S32 * p) @ g64.abs())
    return {name: (x, 1.02 * (ex + u * x.abs())) for name, x, ex in (("dq", dq, edq), ("dk", dk, edk), ("dv", dv, edv))}


CASES = [
    # z, h, hk, n, s, d, window, sinks, layout
    (1, 4, 4, 1500, 1500, 64, 1000, 4, "heads"),
    (1, 8, 2, 1500, 1500, 128, 5000, 0, "tokens"),
    (1, 8, 1, 900, 900, 64, 300, 40, "tokens"),      # lists in parts
    (1, 6, 2, 1200, 1200, 32, 700, 0, "heads"),
    (2, 4, 2, 800, 800, 16, 5000, 3, "tokens"),
    (2, 4, 1, 300, 1500, 128, 900, 5, "heads"),      # the last queries of longer keys
    (1, 4, 4, 3000, 3000, 64, 5000, 0, "heads"),
]


def gradients(q, k, v, do, window, sinks, scale):
    from tattn import window_attention

    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    return torch.autograd.grad(window_attention(*leaves, window, sinks, sm_scale=scale), leaves, do)


@pytest.mark.parametrize("z,h,hk,n,s,d,window,sinks,layout", CASES)
@pytest.mark.parametrize("shift", [9, 13, 16])
def test_gradients_of_small_losses(z, h, hk, n, s, d, window, sinks, layout, shift):
    print("small gradients", z, h, hk, n, s, d, window, sinks, layout, shift, flush=True)
    q, k, v, do = make(z, h, hk, n, s, d, torch.float16, layout, seed=41)
    q, scale = q / 8, 8 * d ** -0.5  # gradients of k as large as they are in training next to their own steps of 2^-24
    do = ((do * 64).round().clamp(-256, 256) / 64) * 2.0 ** -shift  # exact: steps of 2^-22 and more
    want = bounds(q, k, v, do, window, sinks, scale)
    for name, got in zip(("dq", "dk", "dv"), gradients(q, k, v, do, window, sinks, scale)):
        close(name, got, *want[name])


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-35, 3.0])
def test_scales_with_small_losses(d, scale):
    q, k, v, do = make(1, 4, 2, 300, 300, d, torch.float16, seed=42)
    do = (do * 64).round() / 64 * 2.0 ** -15
    want = bounds(q, k, v, do, 200, 4, scale)
    for name, got in zip(("dq", "dk", "dv"), gradients(q, k, v, do, 200, 4, scale)):
        assert got.isfinite().all()
        close(name, got, *want[name])


@pytest.mark.parametrize("d", [32, 64, 128])
def test_rows_without_gradient_and_a_wide_range_of_rows(d):
    """Rows of zeros, of 2^-14 and of 2^4 next to each other, none of it lost where only small rows see a key."""
    q, k, v, do = make(1, 4, 2, 1200, 1200, d, torch.float16, seed=43)
    do = (do * 64).round().clamp(-256, 256) / 64
    do[:, :, 200:900] *= 2.0 ** -14
    do[:, :, 900:1000] = 0
    do[:, :, 1000:] *= 4
    want = bounds(q, k, v, do, 150, 0, d ** -0.5)
    got = dict(zip(("dq", "dk", "dv"), gradients(q, k, v, do, 150, 0, d ** -0.5)))
    for name in got:
        close(name, got[name], *want[name])
    assert (got["dq"][:, :, 900:1000] == 0).all()
    # Keys 300 .. 500 are seen by rows 300 .. 649 alone: relative to those rows' own size.
    small = torch.zeros_like(do)
    small[:, :, 200:900] = do[:, :, 200:900]
    alone = bounds(q, k, v, small, 150, 0, d ** -0.5)
    for name in ("dk", "dv"):
        close(name + " of small rows", got[name][:, :, 300:500], *(t[:, :, 300:500] for t in alone[name]))


@pytest.mark.parametrize("d", [32, 64, 128])
def test_small_gradients_of_values_far_above_one(d):
    """Values of up to 400 with gradients of 2^-12: what is scaled up stays finite."""
    q, k, v, do = make(1, 2, 2, 300, 300, d, torch.float16, seed=44)
    v = (v * 100).clamp(-400, 400)
    do = (do * 64).round() / 64 * 2.0 ** -12
    want = bounds(q, k, v, do, 100, 4, d ** -0.5)
    for name, got in zip(("dq", "dk", "dv"), gradients(q, k, v, do, 100, 4, d ** -0.5)):
        assert got.isfinite().all()
        close(name, got, *want[name])


@pytest.mark.parametrize("window", [2, 100, 5000])
@pytest.mark.parametrize("d", [16, 32, 64, 128])
def test_small_gradients_of_values_near_the_largest(d, window):
    """Values of 60,000 either way, along the gradients: dS of their size is not scaled past float16's largest."""
    q, k, v, do = make(1, 4, 2, 400, 400, d, torch.float16, seed=45)
    sign = torch.where(torch.arange(400, device=DEV) % 3 == 0, 1.0, -1.0)[None, None, :, None]
    v = (60000 * sign).expand_as(v).to(torch.float16).contiguous()
    v[:, :, 300:] /= 1024  # ordinary ones
    do = torch.full_like(do, 2.0 ** -12)
    do[:, :, 100:150] *= 2.0 ** -3
    want = bounds(q, k, v, do, window, 4, d ** -0.5)
    for name, got in zip(("dq", "dk", "dv"), gradients(q, k, v, do, window, 4, d ** -0.5)):
        assert got.isfinite().all(), name
        close(name, got, *want[name])
