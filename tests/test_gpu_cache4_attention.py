"""cache4_attention on the GPU against float64 attention over the values that the cache's bytes stand for, and the serving
path as a whole: pages, norms with rotation, the cache, prompts and single tokens.

Bound, as for attention in general (u: half a step of the element type; f = 2^-25 in float16, the step of small
probabilities; e = (d + 4) 2^-24 sum |q k| scale + 2^-20, the float32 score and the exponential):
  |error| <= sum_j p_j |v_j| (2u + 2e + keys 2^-24) + f sum_j |v_j| + u |o|, times 1.02 for second order."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
LEVELS = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from tattn import hip_available

    assert hip_available(DEV), "libtattn_hip.so did not load or the device is not a gfx950"


def values(cache, table, keys):
    """K, V [kv_heads, keys, d] in float64 of the tokens `keys` of one request, from the cache's bytes."""
    page = cache.page_size
    at, row = table[keys // page].long(), keys % page
    c = cache.codes[at, :, :, row].int()
    x = LEVELS.to(DEV)[torch.stack((c & 15, c >> 4), -1).flatten(-2)]
    e = cache.scales[at, :, :, row].double()
    unit = torch.where(e == 255, math.nan, torch.exp2(e - 127))
    x = (x.unflatten(-1, (-1, 32)) * unit[..., None]).flatten(-2)
    return x[:, :, 0].transpose(0, 1), x[:, :, 1].transpose(0, 1)


def attend(q, k, v, scale):
    """One request: q [h, d], k, v [hk, keys, d]; (o, bound)."""
    u = torch.finfo(q.dtype).eps / 2
    f = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    h, d = q.shape
    k, v = (t.repeat_interleave(h // k.shape[0], 0) for t in (k, v))
    qd = q.double()[:, None]
    p = torch.softmax((qd * k).sum(-1) * scale, -1)
    e = (d + 4) * 2.0 ** -24 * (qd * k).abs().sum(-1).amax(-1) * abs(scale) + 2.0 ** -20
    o = (p[..., None] * v).sum(1)
    bound = (p[..., None] * v.abs()).sum(1) * (2 * u + 2 * e + k.shape[1] * 2.0 ** -24)[:, None] + f * v.abs().sum(1) + u * o.abs()
    return o, 1.02 * bound + torch.finfo(q.dtype).smallest_normal * u


def check(label, got, q, cache, tables, lens, window, sinks, scale, valid=None):
    held = tables.shape[1] * cache.page_size
    worst = 0.0
    for r, n in enumerate(lens.tolist()):
        n = min(max(n, 0), held)
        j = torch.arange(n, device=DEV)
        if window:
            j = j[(j >= n - window) | (j < sinks)]
        pages = tables[r][j // cache.page_size]
        j = j[(pages >= 0) & (pages < cache.pages)]
        if not len(j):
            assert (got[r] == 0).all(), f"{label}: request {r} sees nothing"
            continue
        o, bound = attend(q[r], *values(cache, tables[r], j), scale)
        assert torch.equal(o.isnan(), got[r].isnan()), f"{label}: request {r}"
        err = ((got[r].double() - o).abs() / bound).nan_to_num(0)
        worst = max(worst, err.max().item())
    print(f"{label}: {worst:.2f} of the bound", flush=True)
    assert worst <= 1, label


def make(r, longest, h, hk, d, page, dtype, seed=0, spare=2):
    from tattn import Cache4

    g = torch.Generator().manual_seed(seed + r + longest)
    lens = torch.randint(1, longest + 1, (r,), generator=g, dtype=torch.int32)
    special = [longest, 0, 1, page, longest + 5000, -3]
    for i in range(min(r, len(special))):
        lens[i] = special[i]
    width = (longest + page - 1) // page
    pages = r * width + spare
    tables = torch.randperm(pages, generator=g)[:r * width].view(r, width).to(torch.int32)
    codes = torch.randint(0, 256, (pages, hk, 2, page, d // 2), generator=g, dtype=torch.uint8)
    scales = torch.randint(122, 128, (pages, hk, 2, page, d // 32), generator=g, dtype=torch.uint8)
    q = torch.randn(r, h, d, generator=g).to(DEV, dtype)
    return q, Cache4(codes.to(DEV), scales.to(DEV), dtype), tables.to(DEV), lens.to(DEV)


CASES = [
    # requests, longest, h, hk, d, page, window, sinks, dtype
    (1, 1, 1, 1, 32, 16, 0, 0, torch.float16),
    (6, 40, 4, 4, 64, 16, 0, 0, torch.bfloat16),
    (7, 200, 8, 1, 128, 32, 0, 0, torch.float16),
    (3, 333, 12, 4, 32, 64, 0, 0, torch.bfloat16),
    (9, 500, 16, 2, 128, 16, 100, 4, torch.bfloat16),
    (6, 700, 6, 2, 64, 128, 33, 40, torch.float16),
    (6, 300, 33, 1, 64, 16, 0, 0, torch.float16),       # more than 32 heads to a key head
    (6, 150, 80, 1, 128, 16, 64, 1, torch.bfloat16),
    (1, 9000, 4, 1, 128, 16, 0, 0, torch.bfloat16),     # many parts
    (2, 20000, 8, 2, 64, 64, 0, 0, torch.float16),
    (300, 130, 4, 2, 128, 16, 0, 0, torch.float16),     # many short requests
    (6, 2000, 4, 2, 32, 1024, 1500, 700, torch.bfloat16),
    (6, 600, 4, 2, 128, 16, 1, 0, torch.float16),
    (6, 600, 4, 2, 128, 16, 100000, 3, torch.float16),
]


@pytest.mark.parametrize("r,longest,h,hk,d,page,window,sinks,dtype", CASES)
def test_matches_float64_over_the_held_values(r, longest, h, hk, d, page, window, sinks, dtype):
    from tattn import cache4_attention

    print("cache4_attention", r, longest, h, hk, d, page, window, sinks, dtype, flush=True)
    q, cache, tables, lens = make(r, longest, h, hk, d, page, dtype)
    got = cache4_attention(q, cache, tables, lens, window=window or None, sinks=sinks)
    assert got.dtype == dtype and got.shape == q.shape
    check("o", got, q, cache, tables, lens, window, sinks, d ** -0.5)
    assert torch.equal(got, cache4_attention(q, cache, tables, lens, window=window or None, sinks=sinks))


@pytest.mark.parametrize("d,page", [(64, 16), (128, 64)])
def test_pages_outside_the_window_and_outside_the_cache(d, page):
    """Page numbers of pages without a seen token may be anything; a seen token on a page that is not the cache's is hidden."""
    from tattn import cache4_attention

    q, cache, tables, lens = make(8, 1000, 8, 2, d, page, torch.float16, seed=4)
    clean = cache4_attention(q, cache, tables, lens, window=200, sinks=5)
    stale = tables.clone()
    at = torch.arange(tables.shape[1], device=DEV)[None] * page
    n = lens.clamp(0, tables.shape[1] * page)[:, None]
    unseen = ((at + page <= n - 200) & (at >= 5)) | (at >= n)
    garbage = torch.tensor([-1, cache.pages, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=DEV)
    stale[unseen] = garbage[torch.arange(int(unseen.sum()), device=DEV) % 4]
    assert unseen.any() and torch.equal(cache4_attention(q, cache, stale, lens, window=200, sinks=5), clean)
    holes = tables.clone()
    holes[:, 1::3] = garbage[torch.arange(holes[:, 1::3].shape[1], device=DEV) % 4]
    got = cache4_attention(q, cache, holes, lens)
    check("holes", got, q, cache, holes, lens, 0, 0, d ** -0.5)
    holes[:] = -1
    assert (cache4_attention(q, cache, holes, lens) == 0).all()


def test_blocks_of_nan_reach_those_who_see_them():
    from tattn import cache4_attention

    q, cache, tables, lens = make(6, 400, 4, 2, 128, 16, torch.bfloat16, seed=6)
    lens[:] = torch.tensor([400, 390, 100, 37, 5, 200])
    cache.scales.view(cache.pages, 2, 2, 16, 4)[tables[0, 3].long(), 1, 0, 7, 2] = 255   # a key of request 0, head 1
    cache.scales[tables[1, 24].long(), 0, 1, 9, 0] = 255   # a value of request 1 behind its length (24 * 16 + 9 = 393)
    cache.scales[tables[2, 2].long(), 0, 1, 1, 3] = 255    # a value of request 2, head 0
    got = cache4_attention(q, cache, tables, lens)
    assert got[0, 2:].isnan().all() and not got[0, :2].isnan().any() and not got[1].isnan().any()
    assert got[2, :2, 96:].isnan().all() and not got[2, :2, :96].isnan().any() and not got[3:].isnan().any()
    check("nan", got, q, cache, tables, lens, 0, 0, 128 ** -0.5)
    windowed = cache4_attention(q, cache, tables, lens, window=60, sinks=2)
    assert not windowed[0].isnan().any()


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
def test_scales_and_strides(scale):
    from tattn import cache4_attention

    q, cache, tables, lens = make(6, 300, 8, 4, 64, 32, torch.float16, seed=7)
    wide = torch.zeros(6, 12, 64, dtype=torch.float16, device=DEV)
    wide[:, 2:10] = q
    table = torch.full((6, tables.shape[1] + 3), -1, dtype=torch.int32, device=DEV)
    table[:, :-3] = tables
    got = cache4_attention(wide[:, 2:10], cache, table[:, :-3], lens, sm_scale=scale)
    check("o", got, q, cache, tables, lens, 0, 0, scale)
    flat = torch.zeros(q.numel() + 1, dtype=torch.float16, device=DEV)
    flat[1:] = q.flatten()
    assert torch.equal(cache4_attention(flat[1:].view_as(q), cache, table, lens, sm_scale=scale), got)


def test_offsets_beyond_32_bits():
    """A cache of 4.5 GiB of codes: tokens written, read and attended over on its last pages."""
    from tattn import Cache4, cache4_attention, cache4_read, cache4_write

    pages, page, hk, d = 36900, 128, 8, 128
    codes = torch.empty((pages, hk, 2, page, d // 2), dtype=torch.uint8, device=DEV)
    scales = torch.empty((pages, hk, 2, page, d // 32), dtype=torch.uint8, device=DEV)
    assert codes.numel() > 1 << 32
    cache = Cache4(codes, scales, torch.bfloat16)
    g = torch.Generator().manual_seed(0)
    kv = torch.randn(300, 2, hk, d, generator=g).to(DEV, torch.bfloat16)
    tables = torch.tensor([[pages - 1, pages - 3, pages // 2]], dtype=torch.int32, device=DEV)
    at = torch.arange(300, device=DEV)
    slots = tables[0][at // page].long() * page + at % page
    cache4_write(cache, kv[:, 0], kv[:, 1], slots)
    k, v = values(cache, tables[0], at)
    rk, rv = cache4_read(cache, slots)
    assert torch.equal(rk.transpose(0, 1).double(), k) and torch.equal(rv.transpose(0, 1).double(), v)
    assert ((k - kv[:, 0].transpose(0, 1).double()).abs() <= 0.25 * kv.double().abs().amax()).all()
    q = torch.randn(1, 16, d, generator=g).to(DEV, torch.bfloat16)
    lens = torch.tensor([300], dtype=torch.int32, device=DEV)
    check("far", cache4_attention(q, cache, tables, lens), q, cache, tables, lens, 0, 0, d ** -0.5)


def test_nobody_and_nothing():
    from tattn import cache4_attention

    q, cache, tables, lens = make(3, 50, 4, 2, 64, 16, torch.float16)
    assert cache4_attention(q[:0], cache, tables[:0], lens[:0]).shape == (0, 4, 64)
    assert (cache4_attention(q, cache, tables[:, :0], lens) == 0).all()
    assert (cache4_attention(q, cache, tables, torch.zeros_like(lens)) == 0).all()


def test_two_captured_graphs_with_parts_follow_lengths_and_tables():
    from tattn import cache4_attention

    sets = [make(2, 6000, 8, 2, 128, 16, torch.bfloat16, seed=s) for s in (1, 2)]
    graphs, outs = [], []
    for args in sets:
        cache4_attention(*args)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(cache4_attention(*args))
        graphs.append(graph)
    for step in range(3):
        for q, cache, tables, lens in sets:
            lens[:] = torch.tensor([17 + 2500 * step, 5999 - 700 * step])
            tables.copy_(tables.flip(1))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for args, o in zip(sets, outs):
            assert torch.equal(o, cache4_attention(*args))


def test_another_stream():
    from tattn import cache4_attention

    args = make(4, 3000, 8, 2, 128, 16, torch.float16)
    want = cache4_attention(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = cache4_attention(*args)
    side.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("d,dtype,window,sinks", [(64, torch.float16, 0, 0), (128, torch.bfloat16, 48, 4)])
def test_a_serving_run(d, dtype, window, sinks):
    """Three requests: prompts of unequal lengths, then single tokens, then a second prompt chunk over the cached prefix. Every
    step: page_tables, qk_norm_rope at the tokens' positions, cache4_write, attention. Checked against float64 attention over
    what the cache holds for each request."""
    from tattn import Cache4, cache4_attention, cache4_read, cache4_write, page_tables, qk_norm_rope, window_attention

    h, hk, page, r = 8, 2, 16, 3
    g = torch.Generator().manual_seed(d)
    cache = Cache4.empty(64, page, hk, d, dtype=dtype, device=DEV)
    free = torch.randperm(64, generator=g).to(DEV, torch.int32)
    tables = torch.full((r, 20), -1, dtype=torch.int32, device=DEV)
    lens = torch.zeros(r, dtype=torch.int32, device=DEV)
    angle = torch.arange(400, dtype=torch.float64)[:, None] * 100.0 ** (-torch.arange(d // 2, dtype=torch.float64) / (d // 2))
    cos, sin = angle.cos().float().to(DEV), angle.sin().float().to(DEV)
    qw, kw = ((1 + 0.1 * torch.randn(d, generator=g)).to(DEV, dtype) for _ in range(2))
    seen = window or 10 ** 6
    kept = []  # per step: what was written
    for step, counts in enumerate([[70, 33, 1], [1, 1, 1], [1, 0, 1], [20, 50, 3]]):
        new = torch.tensor(counts, dtype=torch.int32, device=DEV)
        tokens = sum(counts) + 2  # a padded batch
        slots, positions, starts, taken = page_tables(lens, new, tables, free, page, tokens)
        assert starts.tolist() == [0, counts[0], counts[0] + counts[1], sum(counts)]
        proj = torch.randn(1, tokens, h + 2 * hk, d, generator=g).to(DEV, dtype)
        q, k, v = (t.transpose(1, 2) for t in proj.split([h, hk, hk], 2))
        q, k = qk_norm_rope(q, k, qw, kw, cos, sin, positions)
        cache4_write(cache, k[0].transpose(0, 1), v[0].transpose(0, 1), slots)
        lens += new
        free = free[int(taken):]
        at = starts.tolist()
        for i in range(r):
            if counts[i] == 0:
                continue
            n = int(lens[i])
            j = torch.arange(n, device=DEV)
            held = values(cache, tables[i], j)
            mine = q[0, :, at[i]:at[i + 1]]  # [h, count, d]
            if counts[i] == 1:
                batch = q[0, :, at[i]:at[i + 1]].transpose(0, 1)
                got = cache4_attention(batch, cache, tables[i:i + 1], lens[i:i + 1], window=window or None, sinks=sinks)
            else:  # a prompt chunk attends over what the cache holds, its own tokens included
                where = tables[i][j // page].long() * page + j % page
                ck, cv = cache4_read(cache, where)
                got = window_attention(mine[None], ck.transpose(0, 1)[None], cv.transpose(0, 1)[None], seen, sinks)
                got = got[0].transpose(0, 1)
            for c in range(counts[i]):
                p = n - counts[i] + c
                vis = (j <= p) & ((p - j < seen) | (j < sinks))
                o, bound = attend(mine[:, c], held[0][:, vis], held[1][:, vis], d ** -0.5)
                assert ((got[c].double() - o).abs() <= bound).all(), (step, i, c)
        kept.append(counts)
    assert lens.tolist() == [sum(c[i] for c in kept) for i in range(r)]
