"""cross_attention on the GPU against materialised float64 attention: outputs, gradients, lengths, layouts, garbage behind
the lengths, parts, graphs.

Bounds, element by element, from the roundings the kernels make (u: half a step of the element type, s = 2^-24 of float32,
f = 2^-25 in float16, where probabilities below its normal range are rounded to steps of 2^-24; 0 in bfloat16). A score is a
float32 sum of D products: e = (D + 4) s sum |q k| |scale| + 2^-20 relative in its probability (the rest is the exponential's own
error). float32 has the same terms with u = s. Probabilities are rounded once, relative to a maximum of at least 1, and
divided by the sum of the rounded ones:
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


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def visible(z, n, s, lens):
    end = torch.full((z,), s) if lens is None else lens.cpu().long().clamp(0, s)
    return (torch.arange(s)[None, None] < end[:, None, None]).expand(z, n, s).to(DEV)


def plain(q, k, v, do, see, scale):
    """{name: (value, bound)} in float64 for the keys that `see` [z, n, s] shows, with gradients where do is given."""
    u = torch.finfo(q.dtype).eps / 2
    f = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    z, h, n, d = q.shape
    hk, s = k.shape[1:3]
    g = h // hk
    see = see[:, None]
    any_see = see.any(2)[..., None]  # keys that some query sees
    qd = q.double()
    kd, vd = (t.double().masked_fill(~any_see, 0.0).repeat_interleave(g, 1) for t in (k, v))
    kt, vt = kd.transpose(2, 3).contiguous(), vd.transpose(2, 3).contiguous()
    sc = (qd @ kt) * scale
    e = ((d + 4) * S32 * (qd.abs() @ kt.abs()) * abs(scale)).masked_fill(~see, 0.0).amax(-1, keepdim=True) + 2.0 ** -20
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


F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
TRAIN = [
    # z, h, hk, n, s, d, lens, dtype, layout
    (1, 1, 1, 1, 1, 16, None, F16, "heads"),
    (3, 1, 1, 1, 5, 64, (0, 5, 1), BF16, "heads"),
    (2, 3, 1, 5, 9, 32, None, BF16, "tokens"),
    (2, 4, 2, 33, 31, 64, (31, 17), F16, "heads"),
    (1, 2, 2, 32, 32, 128, None, F16, "tokens"),
    (2, 2, 1, 129, 64, 128, (0, 33), BF16, "tokens"),
    (1, 5, 1, 70, 200, 128, (129,), F16, "tokens"),
    (2, 8, 2, 257, 77, 64, (77, 64), F16, "tokens"),
    (1, 6, 2, 100, 300, 32, (299,), F16, "heads"),
    (1, 7, 1, 200, 130, 16, None, BF16, "heads"),
    (2, 12, 4, 300, 513, 64, (500, 513), BF16, "heads"),
    (1, 2, 1, 1000, 321, 128, (320,), BF16, "heads"),
    (1, 4, 4, 2100, 65, 64, None, F16, "heads"),         # few key blocks: rows in parts
    (1, 16, 1, 300, 40, 128, (33,), F16, "tokens"),
    (1, 32, 2, 1, 3000, 64, (2222,), BF16, "heads"),     # few rows: keys in parts
    (2, 4, 2, 3, 2000, 128, (1999, 40), F16, "tokens"),
    (1, 8, 1, 20, 1100, 16, None, F16, "tokens"),
    (40, 2, 1, 40, 40, 64, None, F16, "heads"),
    (1, 3, 3, 640, 900, 64, (900,), BF16, "tokens"),
    (1, 1, 1, 1, 1, 16, None, F32, "heads"),
    (2, 3, 1, 45, 77, 16, (77, 0), F32, "tokens"),
    (1, 6, 2, 200, 150, 32, (149,), F32, "tokens"),
    (2, 4, 4, 257, 300, 64, None, F32, "heads"),
    (1, 5, 1, 100, 333, 128, (200,), F32, "tokens"),
    (1, 8, 2, 2, 2500, 64, (2049,), F32, "heads"),
    (1, 4, 1, 1100, 33, 128, None, F32, "heads"),
]


@pytest.mark.parametrize("z,h,hk,n,s,d,lens,dtype,layout", TRAIN)
def test_outputs_and_gradients_match_float64(z, h, hk, n, s, d, lens, dtype, layout):
    from tattn import cross_attention

    print("cross", z, h, hk, n, s, d, lens, dtype, layout, flush=True)
    lens = None if lens is None else i32(*lens)
    q, k, v, do = make(z, h, hk, n, s, d, dtype, layout)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o = cross_attention(q, k, v, lens)
    grads = torch.autograd.grad(o, leaves, do)
    assert o.dtype == dtype and o.stride() == q.stride()
    with torch.no_grad():
        want = plain(q, k, v, do, visible(z, n, s, lens), d ** -0.5)
        for name, got in zip(("o", "dq", "dk", "dv"), (o, *grads)):
            close(name, got, *want[name])
        assert torch.equal(cross_attention(q, k, v, lens), o)
    o2 = cross_attention(q, k, v, lens)
    for a, b in zip(torch.autograd.grad(o2, leaves, do), grads):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("n,s", [(1, 300), (40, 300), (300, 90)])
def test_garbage_behind_the_lengths_reaches_nothing(n, s, dtype):
    from tattn import cross_attention

    z, h, hk, d = 4, 4, 2, 64
    lens = i32(0, 1, s - 37, s)
    q, k, v, do = make(z, h, hk, n, s, d, dtype)
    behind = (torch.arange(s, device=DEV) >= lens[:, None])[:, None, :, None]

    def run(fill):
        kk, vv = (t.masked_fill(behind, fill).requires_grad_() for t in (k, v))
        qq = q.clone().requires_grad_()
        o = cross_attention(qq, kk, vv, lens)
        return (o.detach(), *torch.autograd.grad(o, (qq, kk, vv), do))

    want = run(0.0)
    for fill in (math.nan, math.inf, -math.inf, torch.finfo(dtype).max):
        for a, b in zip(run(fill), want):
            assert torch.equal(a, b)
    o, dq, dk, dv = want
    assert not o[0].any() and not dq[0].any()
    for t in (dk, dv):
        assert not t.masked_select(behind).any()


def test_lengths_outside_the_keys_are_clamped():
    from tattn import cross_attention

    q, k, v, _ = make(4, 2, 1, 7, 100, 64, F16)
    a = cross_attention(q, k, v, i32(-5, 101, 1 << 30, 100))
    assert torch.equal(a, cross_attention(q, k, v, i32(0, 100, 100, 100)))


@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.0])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_scales(scale, dtype):
    from tattn import cross_attention

    q, k, v, do = make(1, 4, 2, 70, 100, 64, dtype)
    lens = i32(77)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o = cross_attention(q, k, v, lens, sm_scale=scale)
    grads = torch.autograd.grad(o, leaves, do)
    with torch.no_grad():
        want = plain(q, k, v, do, visible(1, 70, 100, lens), scale)
        for name, got in zip(("o", "dq", "dk", "dv"), (o, *grads)):
            close(name, got, *want[name])


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("n", [1, 200])
def test_scores_that_grow_by_far_more_than_a_tile_can_hold(n, dtype):
    """Each tile's scores exceed all before them, so that every one moves the running max; the last keys win."""
    from tattn import cross_attention

    s, d = 700, 64
    q, k, v, _ = make(2, 2, 1, n, s, d, dtype)
    q = q.abs() * 0 + 1
    k = (torch.arange(s, device=DEV) / 16.0)[None, None, :, None].expand(2, 1, s, d).to(dtype).contiguous()
    lens = i32(s, s - 90)
    o = cross_attention(q, k, v, lens)
    close("o", o, *plain(q, k, v, None, visible(2, n, s, lens), d ** -0.5)["o"])


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_views_that_the_kernels_cannot_read_in_place(dtype):
    """Odd strides, unaligned data, broadcast batches and keys, a transposed head dim."""
    from tattn import cross_attention

    g = torch.Generator().manual_seed(3)

    def rand(*shape):
        return torch.randn(*shape, generator=g).to(DEV, dtype)

    q = rand(2, 6, 4, 67)[..., 1:65].transpose(1, 2)                    # unaligned rows
    cases = [
        (rand(1, 2, 50, 64).expand(2, 2, 50, 64), rand(2, 50, 2, 64).transpose(1, 2)),
        (rand(2, 2, 1, 64).expand(2, 2, 50, 64), rand(2, 2, 64, 50).transpose(2, 3)),
        (rand(2, 2, 99, 64)[:, :, ::2], rand(2, 2, 50, 64).flip(0)),
    ]
    for k, v in cases:
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        do = rand(2, 4, 1, 64).expand(2, 4, 6, 64)
        o = cross_attention(*leaves, i32(50, 33))
        grads = torch.autograd.grad(o, leaves, do)
        with torch.no_grad():
            want = plain(q, k, v, do, visible(2, 6, 50, i32(50, 33)), 0.125)
            for name, got in zip(("o", "dq", "dk", "dv"), (o, *grads)):
                close(name, got, *want[name])


def test_a_key_shared_by_a_batch_gets_the_sum_of_its_gradients():
    from tattn import cross_attention

    q, k, v, do = make(3, 4, 2, 20, 70, 64, BF16)
    k1, v1 = k[:1].clone().requires_grad_(), v[:1].clone().requires_grad_()
    o = cross_attention(q, k1.expand(3, -1, -1, -1), v1.expand(3, -1, -1, -1))
    a = torch.autograd.grad(o, (k1, v1), do)
    kk, vv = (t.detach().expand(3, -1, -1, -1).contiguous().requires_grad_() for t in (k1, v1))
    b = torch.autograd.grad(cross_attention(q, kk, vv), (kk, vv), do)
    for x, y in zip(a, b):
        assert torch.equal(x, y.sum(0, keepdim=True))


def test_nothing_to_see_or_to_do():
    from tattn import cross_attention

    for z, n, s in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        q, k, v, do = (torch.randn(z, 2, m, 64, device=DEV, dtype=F16, requires_grad=True) for m in (n, s, s, n))
        o = cross_attention(q, k, v)
        assert o.shape == q.shape and not o.any()
        for g, t in zip(torch.autograd.grad(o, (q, k, v), do), (q, k, v)):
            assert g.shape == t.shape and not g.any()


@pytest.mark.parametrize("by", [-9, -13, 8])
def test_small_and_large_gradients_in_float16(by):
    """dO far below and above 1: dS is held to the precision of its type, not to its range."""
    from tattn import cross_attention

    q, k, v, do = make(1, 4, 2, 300, 400, 64, F16)
    do = do * 2.0 ** by
    leaves = [t.requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(cross_attention(*leaves, i32(390)), leaves, do)
    with torch.no_grad():
        ref = plain(*(t.double() for t in (q, k, v, do)), visible(1, 300, 400, i32(390)), 0.125)
    for name, got in zip(("dq", "dk", "dv"), grads):
        want = ref[name][0]
        # half a step of the result, a few of the operands, and the steps of 2^-24 that the store itself has
        err, norm = (got.double() - want).norm().item(), want.norm().item()
        bound = 4 * 2.0 ** -11 * norm + 2.0 ** -25 * got.numel() ** 0.5
        print(f"{name}: {err:.3e} of {norm:.3e}, bound {bound:.3e}", flush=True)
        assert err <= bound


@pytest.mark.parametrize("opposed", [False, True])
def test_large_values_in_float16_leave_finite_gradients(opposed):
    """Rows of small dO that see large values. Opposed: the largest dS, 0.5 * 64 * 30,000 * 2^-12 = 234, would pass 65,504 times
    the factor that dO's norm of 2^-9 asks for."""
    from tattn import cross_attention

    q, k, v, do = make(1, 2, 1, 64, 2 if opposed else 96, 64, F16)
    v, do = v * 8000, do * 2.0 ** -12
    if opposed:
        v, do = torch.full_like(v, 30000.0), torch.full_like(do, 2.0 ** -12)
        v[:, :, 1] *= -1
    leaves = [t.requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(cross_attention(*leaves), leaves, do)
    with torch.no_grad():
        ref = plain(*(t.double() for t in (q, k, v, do)), visible(1, 64, v.shape[2], None), 0.125)
    for name, got in zip(("dq", "dk", "dv"), grads):
        assert torch.isfinite(got).all()
        want = ref[name][0]
        # dv holds values near 2^-12 * 32 rows in steps of 2^-24 or less
        assert (got.double() - want).norm() <= 8 * 2.0 ** -11 * want.norm()


@pytest.mark.parametrize("dtype,d", [(F16, 64), (BF16, 128)])
def test_gradients_match_differences(dtype, d):
    """The directional derivative of a loss against the central difference of the float64 attention."""
    from tattn import cross_attention

    q, k, v, do = make(1, 2, 1, 50, 70, d, dtype)
    lens, gen = i32(61), torch.Generator().manual_seed(11)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(cross_attention(*leaves, lens), leaves, do)
    see, h = visible(1, 50, 70, lens), 2.0 ** -12
    with torch.no_grad():
        want = plain(q, k, v, do, see, d ** -0.5)
        for i, g in enumerate(grads):
            way = torch.randn(leaves[i].shape, generator=gen).to(DEV, torch.float64)
            ends = []
            for sign in (1, -1):
                x = [t.double() + (sign * h * way if j == i else 0) for j, t in enumerate(leaves)]
                ends.append((plain(*x, None, see, d ** -0.5)["o"][0] * do.double()).sum())
            numeric, analytic = (ends[0] - ends[1]) / (2 * h), (g.double() * way).sum()
            # the gradients' own bounds, and the difference's third-order term
            bound = (want[("dq", "dk", "dv")[i]][1] * way.abs()).sum() + h * h * 100 * way.norm()
            print(f"{numeric.item():.6f} {analytic.item():.6f} bound {bound.item():.2e}", flush=True)
            assert (numeric - analytic).abs() <= bound


def test_a_captured_step_follows_the_lengths():
    from tattn import cross_attention

    z, h, hk, n, s, d = 3, 4, 2, 65, 300, 64
    q, k, v, do = make(z, h, hk, n, s, d, F16)
    lens = i32(300, 10, 77)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    token = make(z, 8, 2, 1, 3000, 128, BF16)[:3]
    token_lens = i32(3000, 1, 1500)

    def step():
        o = cross_attention(*leaves, lens)
        with torch.no_grad():
            t = cross_attention(*token, token_lens)
        return (t, o.detach(), *torch.autograd.grad(o, leaves, do))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed, values in enumerate([(300, 10, 77), (0, 300, 299), (5, 32, 33), (64, 0, 0)]):
        with torch.no_grad():
            for old, new in zip((q, k, v, do), make(z, h, hk, n, s, d, F16, seed=seed)):
                old.copy_(new)
            lens.copy_(i32(*values))
            token_lens.copy_(i32(*(10 * x for x in values)))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, step()):
            assert torch.equal(a, b)


def test_two_streams_at_once():
    from tattn import cross_attention

    work = []
    for seed in (1, 2):
        q, k, v, do = make(1, 8, 2, 130, 1000, 128, F16, seed=seed)
        work.append(([t.requires_grad_() for t in (q, k, v)], do, make(2, 8, 2, 1, 4000, 128, F16, seed=seed)[:3]))

    def job(leaves, do, token):
        o = cross_attention(*leaves, i32(900))
        with torch.no_grad():
            t = cross_attention(*token, i32(4000, 2500))
        return (o.detach(), t, *torch.autograd.grad(o, leaves, do))

    want = [job(*w) for w in work]
    torch.cuda.synchronize()
    sides, got = [torch.cuda.Stream() for _ in work], [[] for _ in work]
    for _ in range(4):
        for out, w, side in zip(got, work, sides):
            with torch.cuda.stream(side):
                out.append(job(*w))
    torch.cuda.synchronize()
    for outs, ref in zip(got, want):
        for out in outs:
            for a, b in zip(out, ref):
                assert torch.equal(a, b)


def test_lengths_changed_before_the_backward_are_noticed():
    from tattn import cross_attention

    q, k, v, do = make(2, 2, 1, 8, 40, 64, F16)
    lens = i32(40, 10)
    o = cross_attention(q.requires_grad_(), k, v, lens)
    lens.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.backward(do)
