"""cross_attention and prefix_attention where one kernel takes over from another, values that are not finite, rows far apart in
memory, and the operators run after one another as programs use them. Bounds of test_gpu_cross."""

import math

import pytest
import torch
from test_gpu_cross import BF16, DEV, F16, F32, close, i32, make, plain, visible
from test_gpu_prefix import make as make_prefix
from test_gpu_prefix import want_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from tattn import hip_available

    assert hip_available(DEV), "libtattn_hip.so did not load or the device is not a gfx950"


def check(q, k, v, do, lens, scale, flushed=0.0):
    from tattn import cross_attention

    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = cross_attention(*leaves, lens, sm_scale=scale)
    grads = torch.autograd.grad(o, leaves, do)
    with torch.no_grad():
        want = plain(q, k, v, do, visible(q.shape[0], q.shape[2], k.shape[2], lens), scale)
        for name, got in zip(("o", "dq", "dk", "dv"), (o, *grads)):
            close(name, got, want[name][0], want[name][1] + flushed)


# Key counts on both sides of the tiles that stay in LDS, rows of one and several tiles.
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d,s", [(16, 1), (16, 33), (16, 128), (16, 129), (32, 31), (32, 97), (32, 129), (64, 32), (64, 65), (64, 96),
                                 (64, 127), (64, 129), (128, 32), (128, 33), (128, 64), (128, 65), (128, 127), (128, 129)])
@pytest.mark.parametrize("n", [1, 95])
def test_few_keys(n, d, s, dtype):
    print("few", n, d, s, dtype, flush=True)
    q, k, v, do = make(5, 6, 2, n, s, d, dtype, "tokens" if s % 2 else "heads")
    check(q, k, v, do, i32(s, 0, (s + 1) // 2, max(1, s - 1), min(s, 32)), -0.2 if s % 3 else d ** -0.5)


# Rows: one tile, two, the first that are walked together; keys of no tile, part of one, many parts. Slices that do and do not fill eights.
@pytest.mark.parametrize("z,h,hk,n", [(1, 32, 1, 1), (1, 33, 1, 1), (3, 8, 3 + 1, 16), (9, 4, 1, 16), (9, 13, 1, 5), (2, 8, 8, 64), (17, 3, 1, 22)])
@pytest.mark.parametrize("d,s,dtype", [(64, 1000, BF16), (128, 515, F16), (16, 2050, F16), (32, 130, BF16), (64, 333, F32), (128, 97, F32)])
def test_few_rows(z, h, hk, n, d, s, dtype):
    print("rows", z, h, hk, n, d, s, dtype, flush=True)
    q, k, v, do = make(z, h, hk, n, s, d, dtype, "tokens")
    lens = torch.randint(0, s + 1, (z,), generator=torch.Generator().manual_seed(z + n), dtype=torch.int32).to(DEV)
    check(q, k, v, do, lens, d ** -0.5)


# Scores that climb and fall again, over parts, waves and pairs of products: every way the running max can go.
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n,s,d", [(1, 4000, 128), (200, 900, 64), (300, 1200, 128), (70, 120, 32)])
def test_scores_that_climb_and_fall(n, s, d, dtype):
    """Probabilities below 2^-126, the least normal float32, become 0, which is no relative error of theirs: each takes up to 2^-126
    |dP - delta| of dS with it, |dP - delta| < 2 * 128 * 6 * 6 < 2^14 for normal draws below 6, and a gradient's element up to
    2^9 rows or 2^12 keys times |q| < 2^2 or |k| < 2^6 of that: 2^(-126 + 14 + 18) = 2^-94, far below any value that counts."""
    q, k, v, do = make(2, 4, 2, n, s, d, dtype)
    at = torch.arange(s, device=DEV)
    k = (k + (at % 190 / 19.0 - (at % 64 == 5) * 30.0)[:, None]).to(dtype)
    q = (q * 0.25 + 0.5).to(dtype)
    check(q, k, v, do, i32(s, s - 33), 0.3, 2.0 ** -94)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.0, -3.0])
@pytest.mark.parametrize("n,s,d,dtype", [(1, 300, 64, BF16), (40, 1000, 128, F16), (200, 700, 32, F16), (150, 300, 128, BF16), (70, 300, 64, F32),
                                         (5, 50, 16, F16), (70, 120, 64, BF16)])
def test_any_scale(n, s, d, dtype, scale):
    q, k, v, do = make(3, 4, 2, n, s, d, dtype)
    check(q, k, v, do, i32(s, 0, s - 40), scale, 2.0 ** -94)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.0, -3.0])
@pytest.mark.parametrize("members,n", [(5, 3), (40, 1)])
def test_any_scale_behind_a_prefix(members, n, scale):
    from tattn import prefix_attention

    args = make_prefix(2, members, 4, 2, n, 500, 60, 64, BF16)
    lens, prefix_lens = torch.arange(2 * members, dtype=torch.int32, device=DEV) % 61, i32(0, 333)
    got = prefix_attention(*args, lens, prefix_lens, sm_scale=scale)
    close("o", got, *want_of(*args, lens, prefix_lens, scale))


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("n,s,d,dtype", [(1, 300, 64, BF16), (70, 100, 64, F16), (70, 300, 128, F16), (200, 500, 64, F16), (40, 70, 32, F32)])
def test_what_is_not_finite_stays_in_its_row_and_head(n, s, d, dtype, value):
    """A query that is not finite spoils its own row, and dK and dV of its key head; a key spoils the rows of its sequence and head."""
    from tattn import cross_attention

    q, k, v, do = make(3, 4, 2, n, s, d, dtype)
    row = (torch.arange(3)[:, None, None] == 1) & (torch.arange(4)[:, None] == 2) & (torch.arange(n) == n // 2)
    spoilt = q.masked_fill(row[..., None].to(DEV), value)
    leaves = [t.detach().requires_grad_() for t in (spoilt, k, v)]
    o = cross_attention(*leaves)
    dq, dk, dv = torch.autograd.grad(o, leaves, do)
    other = torch.ones(3, 2, dtype=torch.bool)
    other[1, 1] = False
    with torch.no_grad():
        want = plain(q, k, v, do, visible(3, n, s, None), d ** -0.5)
        for name, got, where in (("o", o, ~row), ("dq", dq, ~row), ("dk", dk, other), ("dv", dv, other)):
            close(name, got[where.to(DEV)], *(x[where.to(DEV)] for x in want[name]))
        assert torch.isnan(o[row.to(DEV)]).all()
        v2 = v.clone()
        v2[1, 1, s // 3] = value
        got = cross_attention(q, k, v2)
        heads = torch.ones(3, 4, dtype=torch.bool)
        heads[1, 2:] = False
        close("o", got[heads.to(DEV)], *(x[heads.to(DEV)] for x in want["o"]))
        assert not torch.isfinite(got[1, 2:]).any()


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("h,n,s", [(4, 1, 300), (8, 1, 60), (4, 2, 300), (6, 33, 200)])
def test_heads_that_share_a_query_or_a_gradient(h, n, s, dtype):
    """Heads of one address: queries that all heads read, and the gradient of a sum over heads. Scores reach 2 * 64 * 3 * 3, so that a
    row that is not there would not be of no weight."""
    q, k, v, do = make(3, h, 2, n, s, 64, dtype)
    lens = i32(s, 0, s - 5)
    check(q, k, v, do[:, :1].expand(-1, h, -1, -1), lens, 0.125)
    check(q[:, :1].expand(-1, h, -1, -1), k, v, do, lens, 2.0, 2.0 ** -94)
    check(q[:, :1].expand(-1, h, -1, -1), k, v, do[:1, :1, :1].expand(3, h, n, 64), lens, 0.125)


def test_rows_far_apart():
    """Batches 2^31 elements apart: offsets pass 32 bits."""
    z, h, n, s, d = 2, 2, 70, 200, 64
    whole = torch.empty((1 << 31) + (1 << 22), device=DEV, dtype=BF16)

    def far(t, at):
        x = whole.as_strided(t.shape, (1 << 31, t.shape[2] * d, d, 1), at)
        return x.copy_(t)

    near = make(z, h, h, n, s, d, BF16)
    check(*(far(t, i << 20) for i, t in enumerate(near)), i32(s, 77), 0.125)


def test_a_long_cache_of_many_bytes():
    """Keys of nearly 2^31 bytes in a head: the last of them are read where they are. Larger ones are refused."""
    from tattn import cross_attention

    s, d = (1 << 23) - 300, 128  # rows of 256 bytes; 256 more would pass 2^31
    k, v = (torch.zeros(1, 1, s, d, device=DEV, dtype=BF16) for _ in range(2))
    q = torch.ones(1, 1, 1, d, device=DEV, dtype=BF16)
    k[0, 0, -1] = 1.0
    v[0, 0, -1] = torch.arange(d, device=DEV)
    o = cross_attention(q, k, v, sm_scale=1.0)
    assert torch.equal(o[0, 0, 0], v[0, 0, -1])  # e^128 outweighs all others
    with pytest.raises(RuntimeError, match="2 GiB"):
        cross_attention(q, *(t.new_empty(1, 1, 1, d).expand(1, 1, 1 << 23, d).contiguous() for t in (k, v)))


PREFIX = [
    # groups, members, h, hk, n, prefix, s, d, dtype: more than 32 rows of a group are walked together
    (1, 32, 1, 1, 1, 2100, 40, 64, F16),
    (1, 33, 1, 1, 1, 2100, 40, 64, F16),
    (3, 17, 4, 2, 1, 700, 100, 128, BF16),
    (2, 65, 2, 1, 1, 1300, 33, 32, F16),
    (2, 11, 12, 1, 1, 520, 700, 16, BF16),
    (1, 130, 8, 2, 2, 4097, 20, 128, F16),
    (9, 40, 1, 1, 1, 31, 65, 64, BF16),
]


@pytest.mark.parametrize("groups,members,h,hk,n,p,s,d,dtype", PREFIX)
def test_rows_behind_a_prefix(groups, members, h, hk, n, p, s, d, dtype):
    from tattn import prefix_attention

    print("prefix", groups, members, h, hk, n, p, s, d, dtype, flush=True)
    args = make_prefix(groups, members, h, hk, n, p, s, d, dtype, "tokens")
    gen = torch.Generator().manual_seed(p)
    lens = torch.randint(0, s + 1, (groups * members,), generator=gen, dtype=torch.int32).to(DEV)
    ragged = torch.randint(0, p + 1, (groups,), generator=gen, dtype=torch.int32).to(DEV)
    for prefix_lens in (None, ragged):
        got = prefix_attention(*args, lens, prefix_lens)
        close("o", got, *want_of(*args, lens, prefix_lens, d ** -0.5))
    behind = (torch.arange(p, device=DEV) >= ragged[:, None])[:, None, :, None]
    spoilt = [t.masked_fill(behind, math.nan) for t in args[1:3]]
    assert torch.equal(prefix_attention(args[0], *spoilt, *args[3:], lens, ragged), got)


# ---- one after the other, as programs use them ----------------------------------------------------

def tables(rows, pairs):
    angles = torch.arange(rows, device=DEV, dtype=torch.float64)[:, None] * 100.0 ** (-torch.arange(pairs, device=DEV) / pairs)
    return angles.cos().float(), angles.sin().float()


def turned(x, cos, sin, pos, axes):
    """[z, heads, n, d] in float64, halves paired."""
    at = pos.long()[list(axes)].T  # [n, d / 2]
    pair = torch.arange(len(axes), device=DEV)
    c, s = cos.double()[at, pair], sin.double()[at, pair]
    a, b = x.double().chunk(2, -1)
    return torch.cat((a * c - b * s, b * c + a * s), -1)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_a_layer_over_image_tokens_and_a_text(dtype):
    """Rotated heads that attend to each other's grid and to a padded text, trained: the gradients pass through all of it.

    Every result that goes on is rounded to u, half a step of the type; along the way to a gradient lie at most twelve such
    roundings (rotated q and k, P, O, of both attentions, and backward dS, dQ or dK or dV, the turn back, and their sums), and a
    score of up to 8 turns one of its own into 8 u of its probability; errors of independent signs add no faster than one by one:
    12 + 4 * 8 = 44 u of a gradient's norm."""
    from tattn import cross_attention, qk_rope_axes, window_attention

    z, h, hk, d, side, text = 2, 4, 2, 64, 12, 50
    n = side * side
    q, k, v, do = make(z, h, hk, n, n, d, dtype)
    tq, tk, tv, _ = make(z, h, hk, n, text, d, dtype, "tokens", seed=5)
    lens = i32(50, 21)
    cos, sin = tables(64, d // 2)
    grid = torch.arange(n, device=DEV)
    pos, axes = torch.stack((grid // side, grid % side)).to(torch.int32), (0,) * 16 + (1,) * 16
    leaves = [t.requires_grad_() for t in (q, k, v, tq, tk, tv)]

    def layer(q, k, v, tq, tk, tv):
        rq, rk = qk_rope_axes(q, k, cos, sin, pos, axes)
        return window_attention(rq, rk, v, n) + cross_attention(rq + tq, tk, tv, lens)

    out = layer(*leaves)
    grads = torch.autograd.grad(out, leaves, do)
    big = [t.detach().double().requires_grad_() for t in leaves]
    rq, rk = (turned(t, cos, sin, pos, axes) for t in big[:2])

    def attend(a, b, c, see):
        b, c = (t.repeat_interleave(h // hk, 1) for t in (b, c))
        s = (a @ b.transpose(2, 3).contiguous()) * d ** -0.5
        return torch.softmax(s.masked_fill(~see, -math.inf), -1) @ c

    causal = torch.ones(n, n, device=DEV).tril().bool()
    want = attend(rq, rk, big[2], causal) + attend(rq + big[3], big[4], big[5], visible(z, n, text, lens)[:, None])
    u = torch.finfo(dtype).eps / 2
    for name, got, ref in zip(("out", "dq", "dk", "dv", "dtq", "dtk", "dtv"), (out, *grads),
                              (want, *torch.autograd.grad(want, big, do.double()))):
        err = ((got.double() - ref).norm() / ref.norm()).item()
        print(f"{name}: {err / u:.1f} u", flush=True)
        assert err <= 44 * u, name

    # The same step captured, with leaves of its own, of which no eager graph lives, and replayed between eager steps.
    own = [t.detach().clone().requires_grad_() for t in leaves]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch.autograd.grad(layer(*own), own, do)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o2 = layer(*own)
        held = (o2.detach(), *torch.autograd.grad(o2, own, do))
    for seed in range(3):
        with torch.no_grad():
            lens.copy_(i32(7 * seed, 50 - seed))
            for t in (leaves[0], own[0]):
                t.copy_(make(z, h, hk, n, n, d, dtype, seed=20 + seed)[0])
        graph.replay()
        torch.cuda.synchronize()
        o3 = layer(*leaves)
        for a, b in zip(held, (o3.detach(), *torch.autograd.grad(o3, leaves, do))):
            assert torch.equal(a, b)


def test_decoding_behind_a_prefix_with_an_encoder():
    """Steps of sequences behind one prompt: the new token's heads are turned, its key and value go into the sequence's own cache,
    it attends to the prompt and to its own tokens, then to encoder states; as one captured step, against the same eagerly and
    against float64."""
    from tattn import cross_attention, prefix_attention, qk_rope_axes

    z, h, hk, d, p, room, states = 40, 8, 2, 64, 300, 16, 77
    _, pk, pv, own_k, own_v = make_prefix(1, z, h, hk, 1, p, room, d, BF16)
    _, ek, ev, _ = make(z, h, hk, 1, states, d, BF16, "tokens")
    elens = torch.randint(0, states + 1, (z,), generator=torch.Generator().manual_seed(1), dtype=torch.int32).to(DEV)
    cos, sin = tables(512, d // 2)
    axes = tuple(i % 2 for i in range(d // 2))
    q, k, v, _ = make(z, h, hk, 1, 1, d, BF16)
    lens = torch.zeros(z, dtype=torch.int32, device=DEV)
    batch = torch.arange(z, device=DEV)

    def step():
        pos = torch.stack((lens + p, lens // 2)).to(torch.int32)[..., None]  # [axes, batch, 1]
        rq, rk = qk_rope_axes(q, k, cos, sin, pos, axes)
        at = lens.long()
        own_k[batch, :, at] = rk[:, :, 0]
        own_v[batch, :, at] = v[:, :, 0]
        lens.add_(1)
        a = prefix_attention(rq, pk, pv, own_k, own_v, lens)
        return rq, a, cross_attention(a, ek, ev, elens)

    with torch.no_grad():
        step()
        lens.zero_()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        lens.zero_()
        for i in range(room):
            for old, new in zip((q, k, v), make(z, h, hk, 1, 1, d, BF16, seed=100 + i)[:3]):
                old.copy_(new)
            caches = own_k.clone(), own_v.clone(), lens.clone()
            graph.replay()
            torch.cuda.synchronize()
            after = [t.clone() for t in (*held, own_k, own_v, lens)]
            for old, new in zip((own_k, own_v, lens), caches):
                old.copy_(new)
            eager = step()
            for a, b in zip(after, (*eager, own_k, own_v, lens)):
                assert torch.equal(a, b)
            rq, a, c = eager
            close("prefix", a, *want_of(rq, pk, pv, own_k, own_v, lens, None, d ** -0.5))
            close("states", c, *plain(a, ek, ev, None, visible(z, 1, states, elens), d ** -0.5)["o"])
        assert lens.eq(room).all()
