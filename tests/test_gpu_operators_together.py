"""The operators around attention as a training step uses them, one after the other, and from several streams.

A chain is checked at its seams: what each operator made of what it was given, against float64 and within the bounds that the
operators' own tests derive, so that no bound has to cover two of them."""

import pytest
import test_gpu_norm_rope as norm
import test_gpu_window as win
import torch

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from tattn import hip_available

    assert hip_available(DEV), "libtattn_hip.so did not load or the device is not a gfx950"


def block(z, n, h, hk, d, dtype, seed=0):
    """(projection [z, n, (h + 2 hk) d], weights, tables, positions, output gradient [z, n, h d])."""
    g = torch.Generator().manual_seed(seed)
    proj = torch.randn(z, n, (h + 2 * hk) * d, generator=g).to(DEV, dtype)
    qw, kw = ((1 + 0.2 * torch.randn(d, generator=g)).to(DEV) for _ in range(2))
    a = torch.rand(n + 7, d // 2, generator=g, dtype=torch.float64) * 6.28
    pos = torch.stack([torch.randperm(n + 7, generator=g)[:n] for _ in range(z)]).to(DEV, torch.int32)
    return proj, qw, kw, a.cos().float().to(DEV), a.sin().float().to(DEV), pos, torch.randn(z, n, h * d, generator=g).to(DEV, dtype)


def run(proj, qw, kw, cos, sin, pos, h, hk, d, window, sinks, seams=None):
    from tattn import qk_norm_rope, window_attention

    z, n = proj.shape[:2]
    q, k, v = (t.transpose(1, 2) for t in proj.view(z, n, h + 2 * hk, d).split([h, hk, hk], 2))
    qr, kr = qk_norm_rope(q, k, qw, kw, cos, sin, pos)
    o = window_attention(qr, kr, v, window, sinks)
    if seams is not None:
        seams.extend((q, k, v, qr, kr, o))
        for t in seams:
            t.retain_grad()
    return o.transpose(1, 2).reshape(z, n, h * d)


@pytest.mark.parametrize("z,n,h,hk,d,window,sinks,dtype", [
    (1, 1, 2, 1, 64, 4, 0, torch.float16),
    (2, 130, 6, 2, 64, 33, 3, torch.bfloat16),
    (1, 301, 4, 4, 128, 90, 0, torch.float16),
    (1, 150, 5, 1, 32, 40, 6, torch.float32),
])
def test_a_training_step(z, n, h, hk, d, window, sinks, dtype):
    """Slices of one projection: norm, rotation, attention, and back to the projection and both weights."""
    proj, qw, kw, cos, sin, pos, do = block(z, n, h, hk, d, dtype)
    for t in (proj, qw, kw):
        t.requires_grad_()
    seams = []
    run(proj, qw, kw, cos, sin, pos, h, hk, d, window, sinks, seams).backward(do)
    q, k, v, qr, kr, o = seams
    with torch.no_grad():
        want = win.plain(qr, kr, v, do.view(z, n, h, d).transpose(1, 2), window, sinks, d ** -0.5)
        for name, got in (("o", o), ("dq", qr.grad), ("dk", kr.grad), ("dv", v.grad)):
            win.close(name, got, *want[name])
        for name, x, w, y, wgrad in (("q", q, qw, qr, qw.grad), ("k", k, kw, kr, kw.grad)):
            yw, yb, dx, dxb, dw, dwb = norm.plain(x, w, cos, sin, pos, 1e-6, False, y.grad)
            norm.close(name, y, yw, yb)
            norm.close("d" + name, x.grad, dx, dxb)
            norm.close(f"d{name}_weight", wgrad, dw, dwb)
        parts = torch.cat([t.grad.transpose(1, 2) for t in (q, k, v)], 2)
        assert torch.equal(proj.grad.view(z, n, h + 2 * hk, d), parts)


def test_a_captured_training_step():
    """Forward and backward of the chain in one graph, replayed on new values between eager steps."""
    z, n, h, hk, d = 1, 200, 4, 2, 64
    proj, qw, kw, cos, sin, pos, do = block(z, n, h, hk, d, torch.bfloat16)
    leaves = [t.requires_grad_() for t in (proj, qw, kw)]

    def step():
        o = run(*leaves, cos, sin, pos, h, hk, d, 50, 4)
        return (o.detach(), *torch.autograd.grad(o, leaves, do))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (1, 2, 3):
        new = block(z, n, h, hk, d, torch.bfloat16, seed)
        with torch.no_grad():
            for old, x in zip((proj, qw, kw, cos, sin, pos, do), new):
                old.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, step()):
            assert torch.equal(a, b)


def test_two_streams_at_once():
    """Training steps and split single-token calls issued in turn to two streams: every result is the one of a call by itself."""
    from tattn import window_attention

    z, n, h, hk, d = 1, 500, 8, 2, 128
    work = []
    for seed in (1, 2):
        proj, qw, kw, cos, sin, pos, do = block(z, n, h, hk, d, torch.float16, seed)
        token = win.make(2, 8, 2, 1, 4000, 128, torch.float16, seed=seed)[:3]
        work.append(([t.requires_grad_() for t in (proj, qw, kw)], (cos, sin, pos), do, token))

    def job(leaves, tables, do, token):
        o = run(*leaves, *tables, h, hk, d, 100, 4)
        grads = torch.autograd.grad(o, leaves, do)
        return (o.detach(), *grads, window_attention(*token, 3000, 8, lens=torch.tensor([4000, 2500], dtype=torch.int32, device=DEV)))

    want = [job(*w) for w in work]
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in work]
    got = [[] for _ in work]
    for _ in range(4):
        for out, w, side in zip(got, work, sides):
            with torch.cuda.stream(side):
                out.append(job(*w))
    torch.cuda.synchronize()
    for outs, ref in zip(got, want):
        for out in outs:
            for a, b in zip(out, ref):
                assert torch.equal(a, b)
