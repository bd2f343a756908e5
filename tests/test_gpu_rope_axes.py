"""qk_rope_axes on the GPU against the formulas in float64 and against differences.

Bounds as in test_gpu_norm_rope (s = 2^-24 of float32, results rounded once): with norms its own; without, a turn is two
products and a sum of float32, 4 s (|a cos| + |b sin|), for the gradients too."""

import math

import pytest
import test_gpu_norm_rope as norm
import torch

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
S = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from tattn import hip_available

    assert hip_available(DEV), "libtattn_hip.so did not load or the device is not a gfx950"


def angles(cos, sin, pos, axes, z):
    """Cosines and sines [z, 1, n, d / 2] of every pair, in float64."""
    if pos.dim() == 2:
        pos = pos[:, None].expand(-1, z, -1)
    c = torch.ones(z, pos.shape[2], len(axes), dtype=torch.float64, device=DEV)
    s = torch.zeros_like(c)
    for i, a in enumerate(axes):
        if a >= 0:
            c[..., i], s[..., i] = cos[:, i].double()[pos[a].long()], sin[:, i].double()[pos[a].long()]
    return c[:, None], s[:, None]


def larger(x, c, s, interleaved):
    """|a c| + |b s| of either of a pair."""
    x, c, s = x.abs(), c.abs(), s.abs()
    return torch.maximum(norm.turn(x, c, s, interleaved).abs(), norm.turn(x, c, -s, interleaved).abs())


def plain(x, w, c, s, eps, interleaved, g):
    """(y, bound), (dx, bound), (dw, bound or None) in float64."""
    x, g = x.double(), g.double()
    t, ta = norm.turn(g, c, -s, interleaved), larger(g, c, s, interleaved)
    if w is None:
        return (norm.turn(x, c, s, interleaved), 4 * S * larger(x, c, s, interleaved)), (t, 4 * S * ta), None
    w = w.double()
    r = 1 / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    xr = x * r
    m, ma = (t * w * xr).mean(-1, keepdim=True), (ta * w.abs() * xr.abs()).mean(-1, keepdim=True)
    return ((norm.turn(xr * w, c, s, interleaved), 32 * S * larger(xr * w, c, s, interleaved)),
            (r * (t * w - xr * m), 64 * S * r * (ta * w.abs() + xr.abs() * ma)),
            ((t * xr).sum((0, 1, 2)), 128 * S * (ta * xr.abs()).sum((0, 1, 2))))


def inputs(z, h, hk, n, d, count, dtype, layout, seed, deep=True, wide=False, rows=300):
    q, k, qw, kw, cos, sin, _, gq, gk = norm.inputs(z, h, hk, n, d, dtype, layout, seed, wide, rows)
    g = torch.Generator().manual_seed(seed + 1)
    pos = torch.randint(0, rows, (count, z, n) if deep else (count, n), generator=g, dtype=torch.int32).to(DEV)
    return q, k, qw, kw, cos, sin, pos, gq, gk


def cut(d, *counts):
    out = [a for a, c in enumerate(counts) for _ in range(c)]
    return tuple(out + [-1] * (d // 2 - len(out)))


CASES = [
    # z, h, hk, n, d, axes, positions for each sequence, dtype, layout, interleaved, norms, wide weights
    (1, 1, 1, 1, 16, cut(16, 2, 3, 3), True, torch.float16, "heads", False, False, False),
    (2, 3, 1, 5, 16, cut(16, 8), False, torch.float32, "tokens", True, False, False),
    (3, 5, 2, 17, 32, cut(32, 4, 4, 8), True, torch.bfloat16, "tokens", False, True, True),
    (1, 4, 4, 33, 32, cut(32, 0, 7, 7), True, torch.float16, "heads", True, False, False),      # pairs that are not turned
    (2, 8, 2, 70, 64, cut(64, 8, 12, 12), False, torch.bfloat16, "tokens", False, False, False),
    (1, 7, 3, 129, 64, tuple(i % 3 for i in range(32)), True, torch.float32, "heads", False, True, False),
    (32, 16, 4, 1, 128, cut(128, 16, 24, 24), True, torch.bfloat16, "tokens", False, False, False),
    (2, 6, 6, 257, 128, cut(128, 9, 21, 30, 1), True, torch.float16, "heads", True, True, True),
    (1, 9, 1, 200, 128, tuple(i % 8 for i in range(64)), False, torch.float32, "tokens", True, False, False),
    (4, 12, 4, 300, 128, cut(128, 16, 24, 24), True, torch.bfloat16, "tokens", False, True, False),
    (1, 2, 2, 40, 64, (-1,) * 32, True, torch.float16, "heads", False, False, False),           # none is
]


@pytest.mark.parametrize("z,h,hk,n,d,axes,deep,dtype,layout,interleaved,norms,wide", CASES)
def test_outputs_and_gradients_match_float64(z, h, hk, n, d, axes, deep, dtype, layout, interleaved, norms, wide):
    from tattn import qk_rope_axes

    print("rope_axes", z, h, hk, n, d, dtype, layout, interleaved, norms, flush=True)
    q, k, qw, kw, cos, sin, pos, gq, gk = inputs(z, h, hk, n, d, max(axes + (0,)) + 1, dtype, layout, z * n + d, deep, wide)
    kw_args = dict(q_weight=qw, k_weight=kw, eps=1e-5) if norms else {}
    leaves = [t.requires_grad_() for t in ((q, k, qw, kw) if norms else (q, k))]
    qo, ko = qk_rope_axes(q, k, cos, sin, pos, axes, interleaved, **kw_args)
    assert qo.stride() == q.stride() and qo.dtype == dtype
    got = torch.autograd.grad((qo, ko), leaves, (gq, gk))
    with torch.no_grad():
        c, s = angles(cos, sin, pos, axes, z)
        for i, (name, x, w, g, o) in enumerate((("q", q, qw, gq, qo), ("k", k, kw, gk, ko))):
            y, dx, dw = plain(x, w if norms else None, c, s, 1e-5, interleaved, g)
            norm.close(name, o, *y)
            norm.close("d" + name, got[i], *dx)
            if norms:
                norm.close(f"d{name}_weight", got[2 + i], *dw)
        a, b = qk_rope_axes(q, k, cos, sin, pos, axes, interleaved, **kw_args)
    assert torch.equal(a, qo) and torch.equal(b, ko)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norms", [False, True])
def test_one_axis_is_the_rotation_of_qk_norm_rope(norms, interleaved):
    from tattn import qk_norm_rope, qk_rope_axes

    q, k, qw, kw, cos, sin, pos, _, _ = inputs(2, 4, 2, 50, 64, 1, torch.bfloat16, "tokens", 5)
    if norms:
        a = qk_rope_axes(q, k, cos, sin, pos, (0,) * 32, interleaved, q_weight=qw, k_weight=kw)
        b = qk_norm_rope(q, k, qw, kw, cos, sin, pos[0], interleaved=interleaved)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    else:
        a = qk_rope_axes(q, k, cos, sin, pos, [0] * 32, interleaved)
        c, s = angles(cos, sin, pos, (0,) * 32, 2)
        norm.close("q", a[0], norm.turn(q.double(), c, s, interleaved), 4 * S * larger(q.double(), c, s, interleaved))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("axes", [cut(32, 4, 4, 4), cut(32, 5, 6, 3)])
def test_a_position_outside_the_tables_makes_its_axis_nan_and_nothing_else(axes, interleaved):
    from tattn import qk_rope_axes

    q, k, _, _, cos, sin, pos, _, _ = inputs(1, 2, 2, 6, 32, 3, torch.float16, "heads", 9)
    want, _ = qk_rope_axes(q, k, cos, sin, pos, axes, interleaved)
    bad = pos.clone()
    bad[0, 0, 1], bad[1, 0, 2], bad[2, 0, 4], bad[1, 0, 5] = 300, -1, 2 ** 31 - 1, -2 ** 31
    got, _ = qk_rope_axes(q, k, cos, sin, bad, axes, interleaved)
    out = torch.zeros(6, 16, dtype=torch.bool, device=DEV)
    for n, axis in ((1, 0), (2, 1), (4, 2), (5, 1)):
        out[n] = torch.tensor([a == axis for a in axes], device=DEV)
    out = torch.stack((out, out), -1).flatten(-2) if interleaved else torch.cat((out, out), -1)
    assert torch.isnan(got[:, :, out]).all() and torch.equal(got[:, :, ~out], want[:, :, ~out])


def test_views_that_the_kernels_cannot_read_in_place():
    from tattn import qk_rope_axes

    q, k, _, _, cos, sin, pos, gq, gk = inputs(2, 4, 2, 30, 64, 2, torch.float16, "heads", 7)
    axes = cut(64, 10, 22)
    want = qk_rope_axes(q, k, cos, sin, pos, axes)
    odd = torch.empty(2, 4, 30, 67, device=DEV, dtype=torch.float16)[..., 1:65].copy_(q).requires_grad_()
    turned = k.transpose(2, 3).contiguous().transpose(2, 3).requires_grad_()
    every = torch.stack((pos, pos), 3)[..., 0]
    got = qk_rope_axes(odd, turned, cos.t().contiguous().t(), sin, every, axes)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    dq, dk = torch.autograd.grad(got, (odd, turned), (gq[:, :1].expand(-1, 4, -1, -1), gk))
    c, s = angles(cos, sin, pos, axes, 2)
    norm.close("dk", dk, norm.turn(gk.double(), c, -s, False), 4 * S * larger(gk.double(), c, s, False))
    g1 = gq[:, :1].double().expand(-1, 4, -1, -1)
    norm.close("dq", dq, norm.turn(g1, c, -s, False), 4 * S * larger(g1, c, s, False))


def test_no_tokens():
    from tattn import qk_rope_axes

    q, k = torch.randn(2, 4, 0, 64, device=DEV, requires_grad=True), torch.randn(2, 2, 0, 64, device=DEV, requires_grad=True)
    w = torch.ones(64, device=DEV, requires_grad=True)
    table = torch.ones(0, 32, device=DEV)
    pos = torch.zeros(3, 0, dtype=torch.int32, device=DEV)
    for kw in ({}, dict(q_weight=w, k_weight=w.detach().clone().requires_grad_())):
        qo, ko = qk_rope_axes(q, k, table, table, pos, (0,) * 32, **kw)
        assert qo.shape == q.shape and ko.shape == k.shape
        (qo.sum() + ko.sum()).backward()
    assert q.grad.shape == q.shape and not w.grad.any()


@pytest.mark.parametrize("norms", [False, True])
def test_gradients_match_differences(norms):
    from tattn import qk_rope_axes

    q, k, qw, kw, cos, sin, pos, gq, gk = inputs(1, 2, 2, 20, 32, 3, torch.float32, "heads", 13)
    axes = cut(32, 4, 6, 3)
    kw_args = dict(q_weight=qw, k_weight=kw) if norms else {}
    leaves = [t.requires_grad_() for t in ((q, k, qw, kw) if norms else (q, k))]
    grads = torch.autograd.grad(qk_rope_axes(q, k, cos, sin, pos, axes, **kw_args), leaves, (gq, gk))
    c, s = angles(cos, sin, pos, axes, 1)
    gen, h = torch.Generator().manual_seed(3), 2.0 ** -10
    for i, g in enumerate(grads):
        way = torch.randn(leaves[i].shape, generator=gen).to(DEV, torch.float64)
        ends = []
        with torch.no_grad():
            for sign in (1, -1):
                x = [t.double() + (sign * h * way if j == i else 0) for j, t in enumerate(leaves)]
                y = [plain(t, x[2 + j] if norms else None, c, s, 1e-6, False, o)[0][0] for j, (t, o) in enumerate(((x[0], gq), (x[1], gk)))]
                ends.append((y[0] * gq.double()).sum() + (y[1] * gk.double()).sum())
        numeric, analytic = (ends[0] - ends[1]) / (2 * h), (g.double() * way).sum()
        # float32 results of about 1e-6 of their terms, and the difference's third-order term, below 1e-4 at this step
        scale = (g.double() * way).abs().sum() + gq.abs().sum()
        print(f"{numeric.item():.6f} {analytic.item():.6f}", flush=True)
        assert (numeric - analytic).abs() <= 1e-4 * scale


def test_captured_and_replayed():
    from tattn import qk_rope_axes

    axes = cut(64, 8, 12, 12)
    args = inputs(2, 4, 2, 40, 64, 3, torch.bfloat16, "tokens", 1)
    q, k, qw, kw, cos, sin, pos, gq, gk = args
    leaves = [t.requires_grad_() for t in (q, k, qw, kw)]

    def step():
        y = qk_rope_axes(q, k, cos, sin, pos, axes)
        a = torch.autograd.grad(y, (q, k), (gq, gk))
        y2 = qk_rope_axes(q, k, cos, sin, pos, axes, q_weight=qw, k_weight=kw)
        return [t.detach() for t in (*y, *a, *y2, *torch.autograd.grad(y2, leaves, (gq, gk)))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (2, 3, 4):
        with torch.no_grad():
            for old, new in zip(args, inputs(2, 4, 2, 40, 64, 3, torch.bfloat16, "tokens", seed)):
                old.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, step()):
            assert torch.equal(a, b)


def test_far_positions_and_large_tables():
    """A table whose last rows lie past 2^31 bytes would be 4 GB; here positions reach the end of 1.1 GB."""
    from tattn import qk_rope_axes

    rows, d = 1 << 21, 128
    turn = torch.rand(rows, d // 2, device=DEV) * 2 * math.pi
    cos, sin = turn.cos(), turn.sin()
    q, k = torch.randn(1, 2, 9, d, device=DEV), torch.randn(1, 1, 9, d, device=DEV)
    pos = torch.randint(rows - 1000, rows, (3, 9), dtype=torch.int32, device=DEV)
    axes = cut(d, 16, 24, 24)
    qo, _ = qk_rope_axes(q, k, cos, sin, pos, axes)
    c, s = angles(cos, sin, pos, axes, 1)
    norm.close("q", qo, norm.turn(q.double(), c, s, False), 4 * S * larger(q.double(), c, s, False))
