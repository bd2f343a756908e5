"""window_attention on the GPU against materialised float64 attention: outputs, gradients, lengths, layouts, masked garbage.

Bounds, element by element, from the roundings the kernels make (u: half a step of the element type, s = 2^-24 of
float32, f = 2^-25 in float16, where probabilities below its normal range are rounded to steps of 2^-24; 0 in bfloat16).
A score is a float32 sum of D products: e = (D + 4) s sum |q k| |scale| + 2^-20 relative in its probability (the rest
is the exponential's own error). float32 has the same terms with u = s. Probabilities are rounded once, relative to a
maximum of at least 1, and divided by the sum of the rounded ones:
  dO_row   <= sum_j p_j |v_j| (2u + 2e) + f sum_j |v_j| + u |o|
The backward's P = 2^(S - M) has that sum's error through M, and is rounded once as dV's operand; dS = P (dP - delta) has P's,
that of dP (float32) and of delta = dO . O (from the rounded O), and is rounded once:
  ddS <= P |dP - delta| (2u + 2e) + P (edP + edelta) + f,   ddV <= sum_i (P (2u + 2e) + f) |dO| + u |dV|
  ddQ <= |scale| sum_j ddS |k_j| + u |dQ|, dK alike.
Sums over n terms in float32 add n s times the sum of magnitudes; second-order terms and the store are covered by a factor
1.02."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
S32 = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from tattn import hip_available

    assert hip_available(DEV), "libtattn_hip.so did not load or the device is not a gfx950"


def visible(z, n, s, window, sinks, lens=None):
    end = torch.full((z,), s) if lens is None else lens.cpu().long().clamp(0, s)
    i = (end[:, None] - n + torch.arange(n))[:, :, None]
    j = torch.arange(s)[None, None]
    return ((j <= i) & ((i - j < window) | (j < sinks))).to(DEV)


def plain(q, k, v, do, window, sinks, scale, lens=None):
    """{name: (value, bound)} in float64, with gradients where do is given."""
    u = torch.finfo(q.dtype).eps / 2
    f = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    z, h, n, d = q.shape
    hk, s = k.shape[1:3]
    g = h // hk
    see = visible(z, n, s, window, sinks, lens)[:, None]
    qd, kd, vd = q.double(), k.double().repeat_interleave(g, 1), v.double().repeat_interleave(g, 1)
    kt, vt = kd.transpose(2, 3).contiguous(), vd.transpose(2, 3).contiguous()
    sc = (qd @ kt) * scale
    e = ((d + 4) * S32 * (qd.abs() @ kt.abs()) * abs(scale)).masked_fill(~see, 0.0).amax((-1), keepdim=True) + 2.0 ** -20
    none = ~see.any(-1, keepdim=True)
    p = torch.softmax(sc.masked_fill(~see, -math.inf), -1).masked_fill(none, 0.0)
    o = p @ vd
    eo = (p @ vd.abs()) * (2 * u + 2 * e + s * S32) + f * (see.double() @ vd.abs()) + u * o.abs()
    out = {"o": (o, 1.02 * eo)}
    if do is None:
        return out
    g64 = do.double()
    dp = g64 @ vt
    delta = (g64 * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    edp = (d + 4) * S32 * (g64.abs() @ vt.abs())
    edelta = (g64.abs() * (eo + (d + 4) * S32 * o.abs())).sum(-1, keepdim=True)
    ep = p * (2 * u + 2 * e)
    eds = ep * (dp - delta).abs() + p * (edp + edelta) + f * see

    def t(x):
        return x.transpose(2, 3).contiguous()

    def group(x):
        return x.reshape(z, hk, g, s, d).sum(2)

    dq, edq = ds @ kd * scale, (eds + s * S32 * ds.abs()) @ kd.abs() * abs(scale)
    dk, edk = group(t(ds) @ qd) * scale, group(t(eds + n * g * S32 * ds.abs()) @ qd.abs()) * abs(scale)
    dv, edv = group(t(p) @ g64), group(t(ep + f * see + n * g * S32 * p) @ g64.abs())
    for name, x, ex in (("dq", dq, edq), ("dk", dk, edk), ("dv", dv, edv)):
        out[name] = x, 1.02 * (ex + u * x.abs())
    return out


def close(label, got, want, bound):
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps / 2
    err = (got.double() - want).abs()
    worst = (err / (bound + tiny)).max().item()
    print(f"{label}: largest error {err.max().item():.3e}, {worst:.2f} of its bound", flush=True)
    assert worst <= 1, label


def make(z, h, hk, n, s, d, dtype, layout="heads", seed=0):
    gen = torch.Generator().manual_seed(seed + 7 * n + s + d)

    def one(heads, length):
        t = torch.randn(z, heads, length, d, generator=gen).to(DEV, dtype)
        return t.transpose(1, 2).contiguous().transpose(1, 2) if layout == "tokens" else t

    return one(h, n), one(hk, s), one(hk, s), one(h, n)


TRAIN = [
    # z, h, hk, n, s, d, window, sinks, dtype, layout
    (1, 1, 1, 1, 1, 16, 1, 0, torch.float16, "heads"),
    (2, 3, 1, 5, 5, 32, 2, 1, torch.bfloat16, "heads"),
    (1, 2, 2, 32, 32, 64, 32, 0, torch.float16, "tokens"),
    (2, 4, 2, 33, 33, 64, 7, 2, torch.float16, "heads"),
    (1, 5, 1, 70, 70, 128, 20, 40, torch.bfloat16, "tokens"),
    (1, 8, 2, 257, 257, 128, 64, 4, torch.float16, "tokens"),
    (3, 2, 2, 300, 300, 64, 100, 4, torch.bfloat16, "heads"),
    (1, 6, 2, 300, 300, 32, 31, 0, torch.float16, "tokens"),
    (1, 7, 1, 200, 200, 16, 50, 3, torch.float16, "heads"),
    (2, 12, 4, 513, 513, 64, 96, 5, torch.bfloat16, "tokens"),
    (1, 2, 1, 1000, 1000, 128, 130, 64, torch.bfloat16, "heads"),
    (1, 1, 1, 2100, 2100, 64, 1, 1, torch.float16, "heads"),
    (1, 3, 1, 2100, 2100, 128, 65, 33, torch.float16, "tokens"),
    (1, 1, 1, 600, 600, 32, 5000, 0, torch.float16, "heads"),     # every earlier key
    (1, 2, 1, 600, 600, 64, 100, 5000, torch.bfloat16, "heads"),  # all keys stay
    (2, 4, 2, 40, 200, 64, 30, 4, torch.float16, "heads"),        # the last queries of longer keys
    (1, 4, 4, 1, 150, 128, 20, 10, torch.bfloat16, "tokens"),
    (1, 9, 3, 77, 400, 32, 150, 0, torch.float16, "tokens"),
    (9, 16, 16, 128, 128, 64, 40, 4, torch.float16, "heads"),
    (1, 8, 1, 700, 700, 64, 300, 0, torch.float16, "tokens"),     # few key blocks, long lists: in parts
    (1, 8, 1, 900, 900, 128, 5000, 0, torch.bfloat16, "heads"),
    (1, 16, 1, 500, 500, 32, 200, 70, torch.float16, "heads"),
    (1, 12, 1, 300, 900, 128, 400, 3, torch.bfloat16, "tokens"),
    (1, 32, 1, 100, 100, 16, 100, 0, torch.float16, "tokens"),
    (1, 1, 1, 1, 1, 16, 1, 0, torch.float32, "heads"),
    (2, 3, 1, 45, 45, 16, 9, 2, torch.float32, "tokens"),
    (1, 6, 2, 200, 200, 32, 31, 0, torch.float32, "tokens"),
    (2, 4, 4, 257, 257, 64, 100, 4, torch.float32, "heads"),
    (1, 5, 1, 300, 300, 128, 64, 40, torch.float32, "tokens"),
    (1, 4, 2, 77, 500, 64, 150, 3, torch.float32, "heads"),
    (1, 2, 1, 400, 400, 128, 1000, 0, torch.float32, "heads"),
]


@pytest.mark.parametrize("z,h,hk,n,s,d,window,sinks,dtype,layout", TRAIN)
def test_outputs_and_gradients_match_float64(z, h, hk, n, s, d, window, sinks, dtype, layout):
    from tattn import window_attention

    print("window", z, h, hk, n, s, d, window, sinks, dtype, layout, flush=True)
    q, k, v, do = make(z, h, hk, n, s, d, dtype, layout)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o = window_attention(q, k, v, window, sinks)
    grads = torch.autograd.grad(o, leaves, do)
    assert o.dtype == dtype and o.stride() == q.stride()
    with torch.no_grad():
        want = plain(q, k, v, do, window, sinks, d ** -0.5)
        for name, got in zip(("o", "dq", "dk", "dv"), (o, *grads)):
            close(name, got, *want[name])
        again = window_attention(q, k, v, window, sinks)
    assert torch.equal(again, o)
    o2 = window_attention(q, k, v, window, sinks)
    for a, b in zip(torch.autograd.grad(o2, leaves, do), grads):
        assert torch.equal(a, b)


@pytest.mark.parametrize("window,sinks", [(1, 0), (31, 0), (32, 1), (33, 32), (64, 33), (65, 100), (1000, 0)])
@pytest.mark.parametrize("d", [64, 128])
def test_every_window_edge_at_every_row(window, sinks, d):
    """One value vector per key, so that the output spells out the probabilities: no key too many, none missing."""
    from tattn import window_attention

    n = 160
    q = torch.zeros(1, 2, n, d, device=DEV, dtype=torch.bfloat16)
    see = visible(1, n, n, window, sinks)[0].double()
    want = see / see.sum(-1, keepdim=True)
    for first in range(0, n, d):
        v = torch.zeros(1, 1, n, d, device=DEV, dtype=torch.bfloat16)
        cols = torch.arange(first, min(n, first + d), device=DEV)
        v[0, 0, cols, cols - first] = 1
        o = window_attention(q, torch.zeros_like(v), v, window, sinks)
        u = torch.finfo(torch.bfloat16).eps / 2
        for head in range(2):
            got = o[0, head, :, :len(cols)].double()
            assert ((got - want[:, cols]).abs() <= 1.01 * u * want[:, cols]).all()


@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0])
def test_scales(scale):
    from tattn import window_attention

    q, k, v, do = make(1, 4, 2, 150, 150, 64, torch.float16, seed=3)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o = window_attention(q, k, v, 60, 4, sm_scale=scale)
    grads = torch.autograd.grad(o, leaves, do)
    with torch.no_grad():
        want = plain(q, k, v, do, 60, 4, scale)
    for name, got in zip(("o", "dq", "dk", "dv"), (o, *grads)):
        close(name, got, *want[name])


LENS = [
    # z, h, hk, n, s, d, window, sinks, dtype, layout
    (1, 1, 1, 1, 1, 64, 1, 0, torch.float16, "heads"),
    (5, 4, 4, 1, 100, 64, 30, 4, torch.bfloat16, "heads"),
    (7, 8, 1, 1, 333, 128, 1000, 0, torch.float16, "tokens"),
    (3, 32, 4, 1, 2000, 128, 512, 4, torch.bfloat16, "heads"),
    (2, 6, 2, 5, 900, 64, 3000, 1, torch.float16, "tokens"),
    (1, 16, 2, 1, 9000, 128, 100000, 0, torch.bfloat16, "heads"),
    (1, 64, 1, 2, 700, 32, 200, 70, torch.float16, "heads"),
    (40, 8, 8, 3, 130, 16, 50, 2, torch.bfloat16, "tokens"),
    (5, 6, 2, 1, 300, 64, 90, 4, torch.float32, "heads"),
    (7, 4, 1, 2, 150, 128, 1000, 0, torch.float32, "tokens"),
]


@pytest.mark.parametrize("z,h,hk,n,s,d,window,sinks,dtype,layout", LENS)
def test_lengths_and_garbage_behind_them(z, h, hk, n, s, d, window, sinks, dtype, layout):
    """Every sequence has its own length (0, 1, short of the queries, beyond the cache among them); NaN and infinities behind
    the lengths and before the windows reach nothing, rows without keys are zeros."""
    from tattn import window_attention

    print("lens", z, h, hk, n, s, d, window, sinks, dtype, layout, flush=True)
    q, k, v, _ = make(z, h, hk, n, s, d, dtype, layout, seed=1)
    gen = torch.Generator().manual_seed(z + s)
    lens = torch.randint(1, s + 1, (z,), generator=gen, dtype=torch.int32)
    special = [0, 1, n - 1, s, s + 100, -5]
    for i in range(min(z - 1, len(special))):
        lens[i] = special[i]
    want = plain(q, k, v, None, window, sinks, d ** -0.5, lens)["o"]
    clean = window_attention(q, k, v, window, sinks, lens=lens.to(DEV))
    close("o", clean, *want)
    see = visible(z, n, s, window, sinks, lens).any(1)  # [z, s]: seen by any row
    bad = torch.tensor([math.nan, math.inf, -math.inf], device=DEV, dtype=dtype)
    for t in (k, v):
        fill = bad[torch.arange(s, device=DEV) % 3][None, None, :, None]
        t.copy_(torch.where(see[:, None, :, None], t, fill))
    assert torch.equal(window_attention(q, k, v, window, sinks, lens=lens.to(DEV)), clean)
    empty = ~visible(z, n, s, window, sinks, lens).any(-1)
    assert (clean.transpose(1, 2)[empty] == 0).all()


@pytest.mark.parametrize("d,dtype", [(32, torch.float16), (64, torch.bfloat16), (128, torch.float16), (64, torch.float32)])
def test_garbage_in_keys_that_no_query_sees(d, dtype):
    """The last queries of longer keys: NaN and infinities before the first window (and behind the first keys) change nothing,
    and their gradients are zeros."""
    from tattn import window_attention

    q, k, v, do = make(1, 6, 2, 100, 700, d, dtype, seed=9)
    unseen = ~visible(1, 100, 700, 77, 5)[0].any(0)
    assert 500 < unseen.sum() < 700
    runs = []
    for fill in (0.0, math.nan, math.inf):
        kk, vv = (torch.where(unseen[None, None, :, None], torch.full_like(t, fill), t).requires_grad_() for t in (k, v))
        qq = q.clone().requires_grad_()
        o = window_attention(qq, kk, vv, 77, 5)
        runs.append((o.detach(), *torch.autograd.grad(o, (qq, kk, vv), do)))
    for a, b, c in zip(*runs):
        assert torch.equal(a, b) and torch.equal(a, c)
    assert (runs[1][2][:, :, unseen] == 0).all() and (runs[1][3][:, :, unseen] == 0).all()


def test_lens_of_whole_rows_are_the_plain_call():
    from tattn import window_attention

    q, k, v, _ = make(2, 4, 2, 100, 100, 64, torch.float16)
    a = window_attention(q, k, v, 30, 4)
    b = window_attention(q, k, v, 30, 4, lens=torch.full((2,), 100, dtype=torch.int32, device=DEV))
    assert torch.equal(a, b)


def test_gradients_match_differences():
    """Along a random direction of each input, in float16 steps that the inputs hold exactly."""
    from tattn import window_attention

    q, k, v, do = make(1, 4, 2, 60, 60, 32, torch.float16, seed=5)
    q, k, v = ((t * 256).round().clamp(-512, 512) / 256 for t in (q, k, v))  # steps of 2^-8, at most 2
    leaves = [t.requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(window_attention(*leaves, 20, 3), leaves, do)
    gen = torch.Generator().manual_seed(1)
    h = 2.0 ** -5
    for leaf, grad in zip(leaves, grads):
        way = torch.randint(-1, 2, leaf.shape, generator=gen).to(DEV, torch.float16)

        def value(sign):
            args = [t.detach() + (sign * h * way if t is leaf else 0) for t in leaves]
            return (window_attention(*args, 20, 3).double() * do.double()).sum()

        diff, exact = (value(1) - value(-1)) / (2 * h), (grad.double() * way.double()).sum()
        # Each output is off by up to 3 u |v| near 1 with signs that do not follow the direction: their sum over 4 x 60 x 32
        # of them stays below 6 standard deviations of it; the third-order term is h^2 of the gradient's own size.
        noise = 6 * 3 * torch.finfo(torch.float16).eps / 2 * do.double().norm() / (2 * h)
        size = (grad.double().abs() * way.double().abs()).sum()
        print("difference", diff.item(), "gradient", exact.item(), "noise", noise.item(), flush=True)
        assert abs(diff - exact) <= noise + h * h * size


def test_layouts_copies_and_broadcast_gradients():
    from tattn import window_attention

    gen = torch.Generator().manual_seed(2)
    proj = torch.randn(2, 90, 8 + 4, 64, generator=gen).to(DEV, torch.bfloat16)
    q, k, v = proj[:, :, :8].transpose(1, 2), proj[:, :, 8:10].transpose(1, 2), proj[:, :, 10:].transpose(1, 2)
    want = plain(q, k, v, torch.ones_like(q), 25, 3, 0.125)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = window_attention(*leaves, 25, 3)
    close("o", o.detach(), *want["o"])
    o.sum().backward()  # a gradient of stride 0
    for name, t in zip(("dq", "dk", "dv"), leaves):
        close(name, t.grad, *want[name])
    odd = torch.randn(2 * 8 * 90 * 64 + 1, generator=gen).to(DEV, torch.bfloat16)[1:].view(2, 8, 90, 64)
    assert torch.equal(window_attention(odd, k, v, 25, 3), window_attention(odd.clone(), k, v, 25, 3))
    one = torch.randn(1, 1, 1, 64, generator=gen).to(DEV, torch.bfloat16)
    wide = one.expand(2, 2, 90, 64)  # every key the same row of memory
    assert torch.equal(window_attention(q, wide, v, 25, 3), window_attention(q, wide.contiguous(), v, 25, 3))
    t = k.transpose(2, 3).contiguous().transpose(2, 3)  # d is not the last stride
    assert torch.equal(window_attention(q, t, v, 25, 3), window_attention(q, k, v, 25, 3))


def test_no_queries_no_keys():
    from tattn import window_attention

    q = torch.zeros(2, 4, 0, 64, device=DEV, dtype=torch.float16, requires_grad=True)
    k = torch.zeros(2, 2, 5, 64, device=DEV, dtype=torch.float16, requires_grad=True)
    o = window_attention(q, k, k, 4)
    o.sum().backward()
    assert o.shape == q.shape and (k.grad == 0).all()
    none = torch.zeros(2, 2, 0, 64, device=DEV, dtype=torch.float16)
    with torch.no_grad():
        o = window_attention(torch.ones(2, 4, 1, 64, device=DEV, dtype=torch.float16), none, none, 4,
                             lens=torch.zeros(2, dtype=torch.int32, device=DEV))
    assert (o == 0).all()


@pytest.mark.parametrize("shape", [(1, 4, 2, 90, 90, 64), (1, 2, 1, 700, 700, 128)])
def test_captured_training_step_replays_on_new_values(shape):
    from tattn import window_attention

    q, k, v, do = make(*shape, torch.bfloat16)
    leaves = [t.requires_grad_() for t in (q, k, v)]

    def step():
        o = window_attention(*leaves, 40, 4)
        grads = torch.autograd.grad(o, leaves, do)
        return (o.detach(), *grads)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(3):
        with torch.no_grad():
            for t, x in zip((q, k, v, do), make(*shape, torch.bfloat16, seed=50 + seed)):
                t.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, step()):
            assert torch.equal(a, b)


def test_captured_single_token_follows_its_lengths():
    """Two graphs of split calls, each with a workspace of its own, replayed in turn as the lengths grow."""
    from tattn import window_attention

    sets = [make(2, 8, 2, 1, 3000, 128, torch.float16, seed=i) for i in range(2)]
    lens = torch.tensor([100, 2000], dtype=torch.int32, device=DEV)
    graphs, outs = [], []
    for q, k, v, _ in sets:
        window_attention(q, k, v, 5000, 0, lens=lens)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(window_attention(q, k, v, 5000, 0, lens=lens))
        graphs.append(graph)
    for step in range(3):
        lens += 1 + 300 * step
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (q, k, v, _), o in zip(sets, outs):
            assert torch.equal(o, window_attention(q, k, v, 5000, 0, lens=lens))
