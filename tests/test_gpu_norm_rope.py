"""qk_norm_rope on the GPU against the formulas in float64 and against differences.

Bounds (u = half a step of the element type, s = 2^-24 of float32). A result is rounded once: u |result|, or half the
smallest subnormal. Before that, in float32: r = 1 / sqrt(mean + eps) carries at most 2 s per term of a lane's chain of 16
squares and 4 swaps (halved by the root) and 3 s of the root itself, under 16 s; x r w adds 2 s and the turn 3 s of either
term, so a result is off by at most 32 s (|a cos| + |b sin|). dx = r (u - x r m): 64 s of the sum of its terms'
magnitudes, m being a mean of D products. A weight's gradient is a sum over rows, at most 32 + 8 + 8 + 48 additions
deep for the sizes here: 128 s of the sum of magnitudes."""

import pytest
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


def turn(x, cos, sin, interleaved):
    half = x.shape[-1] // 2
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :half], x[..., half:])
    a, b = a * cos - b * sin, b * cos + a * sin
    return torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)


def plain(x, w, cos, sin, pos, eps, interleaved, g=None):
    """(y, bound of y's float32 error) and with g (dx, its bound, dw, its bound), in float64."""
    x, w, g = (None if t is None else t.double() for t in (x, w, g))
    c, s = (t.double()[pos.long()][:, None] for t in (cos, sin))
    r = 1 / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    out = [turn(x * r * w, c, s, interleaved), 32 * S * turn((x * r * w).abs(), c.abs(), -s.abs(), False)
           if not interleaved else 32 * S * turn((x * r * w).abs(), c.abs(), -s.abs(), True)]
    # a |c| + b |s| for the first of a pair; the second has the other sign of sin in `turn`.
    out[1] = torch.maximum(out[1].abs(), 32 * S * turn((x * r * w).abs(), c.abs(), s.abs(), interleaved).abs())
    if g is not None:
        t = turn(g, c, -s, interleaved)
        ta = torch.maximum(turn(g.abs(), c.abs(), -s.abs(), interleaved), turn(g.abs(), c.abs(), s.abs(), interleaved))
        xr = x * r
        m = (t * w * xr).mean(-1, keepdim=True)
        ma = (ta * w.abs() * xr.abs()).mean(-1, keepdim=True)
        out += [r * (t * w - xr * m), 64 * S * r * (ta * w.abs() + xr.abs() * ma),
                (t * xr).sum((0, 1, 2)), 128 * S * (ta * xr.abs()).sum((0, 1, 2))]
    return out


def close(label, got, want, bound):
    t = got.dtype
    tiny = torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2
    allow = bound + torch.finfo(t).eps / 2 * (want.abs() + bound) + tiny
    over = ((got.double() - want).abs() - allow).max().item()
    print(f"{label}: largest error {(got.double() - want).abs().max().item():.3e}, over its bound by {over:.3e}", flush=True)
    assert over <= 0, label


def inputs(z, h, hk, n, d, dtype, layout, seed, wide=False, rows=300):
    g = torch.Generator().manual_seed(seed)

    def make(heads):
        t = torch.randn(z, heads, n, d, generator=g) * torch.exp2(torch.randint(-4, 5, (z, heads, n, 1), generator=g).float())
        t = t.to(DEV, dtype)
        return t.transpose(1, 2).contiguous().transpose(1, 2) if layout == "tokens" else t

    q, k, gq, gk = make(h), make(hk), make(h), make(hk)
    qw, kw = ((1 + 0.5 * torch.randn(d, generator=g)).to(DEV, torch.float32 if wide else dtype) for _ in range(2))
    a = torch.rand(rows, d // 2, generator=g, dtype=torch.float64) * 6.28
    cos, sin = a.cos().float().to(DEV), a.sin().float().to(DEV)
    pos = torch.randint(0, rows, (z, n), generator=g, dtype=torch.int32).to(DEV)
    return q, k, qw, kw, cos, sin, pos, gq, gk


CASES = [
    # z, h, hk, n, d, dtype, layout, interleaved, wide weights
    (1, 1, 1, 1, 16, torch.float16, "heads", False, False),
    (2, 3, 1, 5, 16, torch.float32, "tokens", True, False),
    (3, 5, 2, 17, 32, torch.bfloat16, "tokens", False, True),
    (1, 4, 4, 33, 32, torch.float16, "heads", True, False),
    (2, 8, 2, 70, 64, torch.bfloat16, "tokens", False, False),
    (1, 7, 3, 129, 64, torch.float32, "heads", False, False),
    (32, 16, 4, 1, 128, torch.bfloat16, "tokens", False, False),
    (2, 6, 6, 257, 128, torch.float16, "heads", True, True),
    (1, 9, 1, 200, 128, torch.float32, "tokens", True, False),
    (4, 12, 4, 500, 128, torch.bfloat16, "tokens", False, False),
]


@pytest.mark.parametrize("z,h,hk,n,d,dtype,layout,interleaved,wide", CASES)
def test_outputs_and_gradients_match_float64(z, h, hk, n, d, dtype, layout, interleaved, wide):
    from tattn import qk_norm_rope

    print("norm_rope", z, h, hk, n, d, dtype, layout, interleaved, wide, flush=True)
    q, k, qw, kw, cos, sin, pos, gq, gk = inputs(z, h, hk, n, d, dtype, layout, z * n + d, wide)
    for t in (q, k, qw, kw):
        t.requires_grad_()
    qo, ko = qk_norm_rope(q, k, qw, kw, cos, sin, pos, eps=1e-5, interleaved=interleaved)
    assert qo.stride() == q.stride() and qo.dtype == dtype
    got = torch.autograd.grad((qo, ko), (q, k, qw, kw), (gq, gk))
    with torch.no_grad():
        for name, x, w, g, o, dx, dw in (("q", q, qw, gq, qo, got[0], got[2]), ("k", k, kw, gk, ko, got[1], got[3])):
            y, yb, wx, wxb, ww, wwb = plain(x, w, cos, sin, pos, 1e-5, interleaved, g)
            close(f"{name}", o, y, yb)
            close(f"d{name}", dx, wx, wxb)
            close(f"d{name}_weight", dw, ww, wwb)
        again = qk_norm_rope(q, k, qw, kw, cos, sin, pos, eps=1e-5, interleaved=interleaved)
        assert torch.equal(again[0], qo) and torch.equal(again[1], ko)


def test_many_rows_share_out_over_workgroups():
    """More rows than one round of the backward's workgroups takes; twice, bit for bit."""
    from tattn import qk_norm_rope

    q, k, qw, kw, cos, sin, pos, gq, gk = inputs(2, 4, 1, 20000, 64, torch.bfloat16, "tokens", 1)
    for t in (q, k, qw, kw):
        t.requires_grad_()
    runs = []
    for _ in range(2):
        out = qk_norm_rope(q, k, qw, kw, cos, sin, pos)
        runs.append(torch.autograd.grad(out, (q, k, qw, kw), (gq, gk)))
    for a, b in zip(*runs):
        assert torch.equal(a, b)
    with torch.no_grad():
        for x, w, g, dx, dw in ((q, qw, gq, runs[0][0], runs[0][2]), (k, kw, gk, runs[0][1], runs[0][3])):
            _, _, wx, wxb, ww, wwb = plain(x, w, cos, sin, pos, 1e-6, False, g)
            close("dx", dx, wx, wxb)
            close("dw", dw, ww, wwb)


def test_gradients_match_differences():
    from tattn import qk_norm_rope

    q, k, qw, kw, cos, sin, pos, gq, gk = inputs(1, 2, 1, 3, 16, torch.float32, "heads", 9)
    q, k = (q / q.norm(dim=-1, keepdim=True) * 4).requires_grad_(), (k / k.norm(dim=-1, keepdim=True) * 4).requires_grad_()
    leaves = (q, k, qw.requires_grad_(), kw.requires_grad_())
    grads = torch.autograd.grad(qk_norm_rope(*leaves, cos, sin, pos), leaves, (gq, gk))
    for leaf, grad in zip(leaves, grads):
        way = torch.randn(leaf.shape, generator=torch.Generator().manual_seed(2)).to(DEV)
        h = 2.0 ** -7

        def value(sign):
            args = [t.detach() + (sign * h * way if t is leaf else 0) for t in leaves]
            a, b = qk_norm_rope(*args, cos, sin, pos)
            return (a.double() * gq.double()).sum() + (b.double() * gk.double()).sum()

        diff = (value(1) - value(-1)) / (2 * h)
        exact = (grad.double() * way.double()).sum()
        # Third-order term h^2 / 6 of values near 1 with gradients near 1, and rounding s / h of their sum.
        scale = (gq.double().abs().sum() + gk.double().abs().sum()) * 2
        print("difference", diff.item(), "gradient", exact.item(), flush=True)
        assert abs(diff - exact) <= scale * (h * h + 8 * S / h)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_positions_shared_default_and_outside_the_table(dtype):
    from tattn import qk_norm_rope

    q, k, qw, kw, cos, sin, pos, gq, gk = inputs(2, 2, 1, 40, 64, dtype, "heads", 3)
    shared = pos[0].contiguous()
    a = qk_norm_rope(q, k, qw, kw, cos, sin, shared)
    b = qk_norm_rope(q, k, qw, kw, cos, sin, shared.expand(2, 40))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    a = qk_norm_rope(q, k, qw, kw, cos, sin)
    b = qk_norm_rope(q, k, qw, kw, cos, sin, torch.arange(40, dtype=torch.int32, device=DEV))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    bad = pos.clone()
    bad[0, 3], bad[1, 7], bad[1, 8] = -1, 300, 2 ** 31 - 1
    a = qk_norm_rope(q, k, qw, kw, cos, sin, pos)
    b = qk_norm_rope(q, k, qw, kw, cos, sin, bad)
    out = torch.zeros(2, 40, dtype=torch.bool, device=DEV)
    out[0, 3] = out[1, 7] = out[1, 8] = True
    for x, y in zip(a, b):
        assert y.transpose(1, 2)[out].isnan().all()
        assert torch.equal(x.transpose(1, 2)[~out], y.transpose(1, 2)[~out])


def test_zero_rows_odd_layouts_and_frozen_weights():
    """Rows of zeros, slices of one projection, a misaligned tensor, broadcast gradients; no gradient for frozen weights."""
    from tattn import qk_norm_rope

    g = torch.Generator().manual_seed(8)
    proj = torch.randn(2, 30, 10, 64, generator=g).to(DEV, torch.bfloat16)
    proj[0, 4] = 0
    q, k = proj[:, :, :6].transpose(1, 2), proj[:, :, 6:8].transpose(1, 2)
    _, _, qw, kw, cos, sin, pos, _, _ = inputs(2, 1, 1, 30, 64, torch.bfloat16, "heads", 4)
    qo, ko = qk_norm_rope(q, k, qw, kw, cos, sin, pos)
    close("q", qo, *plain(q, qw, cos, sin, pos, 1e-6, False)[:2])
    close("k", ko, *plain(k, kw, cos, sin, pos, 1e-6, False)[:2])
    assert (qo[0, :, 4] == 0).all()
    flat = torch.randn(2 * 6 * 30 * 64 + 1, generator=g).to(DEV, torch.bfloat16)[1:].view(2, 6, 30, 64)
    close("misaligned", qk_norm_rope(flat, k, qw, kw, cos, sin, pos)[0], *plain(flat, qw, cos, sin, pos, 1e-6, False)[:2])
    leaf = q.detach().clone().requires_grad_()
    out, _ = qk_norm_rope(leaf, k, qw, kw, cos, sin, pos)
    out.sum().backward()
    want = plain(leaf.detach(), qw, cos, sin, pos, 1e-6, False, torch.ones_like(out))
    close("sum", leaf.grad, want[2], want[3])
    assert qw.grad is None
    wide = torch.zeros(64, 4, device=DEV, dtype=torch.bfloat16)
    wide[:, 1] = qw
    strided, _ = qk_norm_rope(q, k, wide[:, 1], kw, cos, sin, pos)
    assert torch.equal(strided, qo)


def test_captured_forward_and_backward_replay_on_new_values():
    from tattn import qk_norm_rope

    q, k, qw, kw, cos, sin, pos, gq, gk = inputs(2, 4, 2, 50, 128, torch.float16, "tokens", 6)
    leaves = [t.requires_grad_() for t in (q, k, qw, kw)]

    def step():
        out = qk_norm_rope(*leaves, cos, sin, pos)
        grads = torch.autograd.grad(out, leaves, (gq, gk))
        return (*(t.detach() for t in out), *grads)  # no autograd graph outlives the step

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(3):
        new = inputs(2, 4, 2, 50, 128, torch.float16, "tokens", 60 + seed)
        with torch.no_grad():
            for t, x in zip((q, k, qw, kw, cos, sin, pos, gq, gk), new):
                t.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, step()):
            assert torch.equal(a, b)


def test_no_tokens():
    from tattn import qk_norm_rope

    q = torch.zeros(2, 4, 0, 64, device=DEV, dtype=torch.float16, requires_grad=True)
    w = torch.ones(64, device=DEV, dtype=torch.float16, requires_grad=True)
    cos = torch.ones(5, 32, device=DEV)
    qo, ko = qk_norm_rope(q, q, w, w, cos, cos)
    assert qo.shape == q.shape
    qo.sum().backward()
    assert q.grad.shape == q.shape and (w.grad == 0).all()
