"""prefix_attention on the GPU against materialised float64 attention, within the bounds of test_gpu_cross: the prefix and a
sequence's own keys are one list of keys there."""

import math

import pytest
import torch
from test_gpu_cross import BF16, DEV, F16, close, i32, plain

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from tattn import hip_available

    assert hip_available(DEV), "libtattn_hip.so did not load or the device is not a gfx950"


def make(groups, members, h, hk, n, p, s, d, dtype, layout="heads", seed=0):
    gen, z = torch.Generator().manual_seed(seed + p + s), groups * members

    def one(count, heads, length):
        t = torch.randn(count, heads, length, d, generator=gen).to(DEV, dtype)
        return t.transpose(1, 2).contiguous().transpose(1, 2) if layout == "tokens" else t

    return one(z, h, n), one(groups, hk, p), one(groups, hk, p), one(z, hk, s), one(z, hk, s)


def want_of(q, pk, pv, k, v, lens, prefix_lens, scale):
    z, _, n, _ = q.shape
    groups, p, s = pk.shape[0], pk.shape[2], k.shape[2]
    m = z // groups
    first = torch.full((groups,), p) if prefix_lens is None else prefix_lens.cpu().long().clamp(0, p)
    end = lens.cpu().long().clamp(0, s)
    pos = (end[:, None] - n + torch.arange(n))[..., None]
    see = torch.cat(((torch.arange(p)[None, None] < first.repeat_interleave(m)[:, None, None]) & (pos >= 0),
                     torch.arange(s)[None, None] <= pos), 2).to(DEV)
    kk, vv = (torch.cat((a.repeat_interleave(m, 0), b), 2) for a, b in ((pk, k), (pv, v)))
    return plain(q, kk, vv, None, see, scale)["o"]


CASES = [
    # groups, members, h, hk, n, prefix, s, d, lens, prefix lens, dtype, layout
    (1, 1, 1, 1, 1, 1, 1, 64, (1,), None, F16, "heads"),
    (1, 4, 4, 2, 1, 100, 8, 64, (1, 8, 3, 0), None, F16, "heads"),        # a sequence without a token
    (1, 3, 4, 4, 1, 33, 40, 128, (40, 1, 33), (17,), BF16, "tokens"),
    (2, 3, 8, 2, 2, 70, 64, 64, (2, 64, 33, 1, 5, 6), (0, 70), BF16, "heads"),
    (1, 40, 8, 2, 1, 1000, 16, 128, tuple(range(1, 17)) * 2 + (9,) * 8, None, F16, "heads"),
    (3, 5, 6, 3, 5, 200, 300, 32, tuple(range(5, 300, 20)), (200, 199, 3), F16, "tokens"),
    (1, 2, 16, 1, 7, 64, 50, 16, (50, 7), None, BF16, "heads"),
    (1, 69, 4, 1, 3, 5, 900, 64, tuple(range(3, 900, 13)), None, BF16, "tokens"),
    (2, 2, 2, 2, 1, 4000, 3000, 128, (3000, 1, 2222, 64), (4000, 3999), BF16, "heads"),
    (1, 2, 4, 2, 40, 300, 200, 64, (200, 41), None, F16, "heads"),
    (1, 300, 8, 1, 1, 640, 32, 64, (32, 5, 1) * 100, None, F16, "heads"),  # many rows behind one prefix
]


@pytest.mark.parametrize("groups,members,h,hk,n,p,s,d,lens,prefix_lens,dtype,layout", CASES)
def test_matches_float64(groups, members, h, hk, n, p, s, d, lens, prefix_lens, dtype, layout):
    from tattn import prefix_attention

    print("prefix", groups, members, h, hk, n, p, s, d, dtype, layout, flush=True)
    args = make(groups, members, h, hk, n, p, s, d, dtype, layout)
    lens, prefix_lens = i32(*lens), None if prefix_lens is None else i32(*prefix_lens)
    o = prefix_attention(*args, lens, prefix_lens)
    assert o.dtype == dtype and o.stride() == args[0].stride()
    close("o", o, *want_of(*args, lens, prefix_lens, d ** -0.5))
    assert torch.equal(prefix_attention(*args, lens, prefix_lens), o)


@pytest.mark.parametrize("p,s", [(0, 40), (40, 0), (0, 0)])
def test_no_prefix_or_no_keys_of_its_own(p, s):
    from tattn import prefix_attention

    args = make(2, 3, 4, 2, 1, p, s, 64, F16)
    lens = i32(s, 1, s, 0, s, 2)
    o = prefix_attention(*args, lens)
    if s == 0:
        assert o.shape == args[0].shape and not o.any()  # a query is one of its own keys
    else:
        close("o", o, *want_of(*args, lens, None, 0.125))


@pytest.mark.parametrize("fill", [math.nan, math.inf, -math.inf, 60000.0])
@pytest.mark.parametrize("n", [1, 3])
def test_garbage_behind_the_lengths_reaches_nothing(fill, n):
    from tattn import prefix_attention

    q, pk, pv, k, v = make(2, 2, 4, 2, n, 100, 90, 64, F16)
    lens, prefix_lens = i32(3, 90, 33, 0), i32(0, 65)
    want = prefix_attention(q, pk, pv, k, v, lens, prefix_lens)
    behind = (torch.arange(90, device=DEV) >= lens[:, None])[:, None, :, None]
    pre = (torch.arange(100, device=DEV) >= prefix_lens[:, None])[:, None, :, None]
    got = prefix_attention(q, pk.masked_fill(pre, fill), pv.masked_fill(pre, fill), k.masked_fill(behind, fill),
                           v.masked_fill(behind, fill), lens, prefix_lens)
    assert torch.equal(got, want) and torch.isfinite(got).all()


def test_one_prefix_each_is_a_cache_of_prefix_and_own_keys():
    """Within the bounds, the same as window_attention over both laid in one cache."""
    from tattn import prefix_attention, window_attention

    args = make(3, 1, 8, 2, 2, 64, 100, 128, BF16)
    lens = i32(100, 2, 37)
    q, pk, pv, k, v = args
    value, bound = want_of(*args, lens, None, 128 ** -0.5)
    close("prefix", prefix_attention(*args, lens), value, bound)
    close("window", window_attention(q, torch.cat((pk, k), 2), torch.cat((pv, v), 2), 1000, lens=lens + 64), value, bound)


def test_views_that_the_kernels_cannot_read_in_place():
    from tattn import prefix_attention

    q, pk, pv, k, v = make(1, 4, 4, 2, 1, 50, 20, 64, F16)
    lens = i32(20, 1, 7, 13)
    want = prefix_attention(q, pk, pv, k, v, lens)
    odd = torch.empty(4, 4, 1, 67, device=DEV, dtype=F16)[..., 1:65].copy_(q)
    wide = torch.empty(1, 2, 100, 64, device=DEV, dtype=F16)[:, :, ::2].copy_(pk)
    turned = v.transpose(2, 3).contiguous().transpose(2, 3)
    every = torch.stack((lens, lens), 1)[:, 0]
    assert torch.equal(prefix_attention(odd, wide, pv, k, turned, every), want)


def test_a_captured_call_follows_lengths_and_values():
    from tattn import prefix_attention

    args = make(2, 5, 8, 2, 1, 700, 80, 64, BF16)
    lens, prefix_lens = torch.full((10,), 5, dtype=torch.int32, device=DEV), i32(700, 3)
    prefix_attention(*args, lens, prefix_lens)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = prefix_attention(*args, lens, prefix_lens)
    for seed in range(4):
        for old, new in zip(args, make(2, 5, 8, 2, 1, 700, 80, 64, BF16, seed=seed)):
            old.copy_(new)
        lens.copy_(torch.randint(0, 81, (10,), generator=torch.Generator().manual_seed(seed)))
        prefix_lens.copy_(i32(701 * (seed % 2), 350 + seed))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, prefix_attention(*args, lens, prefix_lens))


def test_two_streams_at_once():
    from tattn import prefix_attention

    work = [(*make(1, 20, 8, 2, 1, 2000, 64, 128, F16, seed=s), torch.full((20,), 9 + s, dtype=torch.int32, device=DEV)) for s in (1, 2)]
    want = [prefix_attention(*w) for w in work]
    torch.cuda.synchronize()
    sides, got = [torch.cuda.Stream() for _ in work], [[] for _ in work]
    for _ in range(8):
        for out, w, side in zip(got, work, sides):
            with torch.cuda.stream(side):
                out.append(prefix_attention(*w))
    torch.cuda.synchronize()
    for outs, ref in zip(got, want):
        assert all(torch.equal(o, ref) for o in outs)
