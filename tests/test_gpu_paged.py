"""Page tables and the cache in 4 bits on the GPU: page_tables against a loop over requests, write and
read against the definition of the format in float64 (every result is exact: no tolerances)."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from tattn import hip_available

    assert hip_available(DEV), "libtattn_hip.so did not load or the device is not a gfx950"


# ---- page_tables ---------------------------------------------------------------------------------

def expected_tables(lens, new, tables, free, page, tokens):
    """One request after the other, one token after the other."""
    tables = [list(row) for row in tables]
    width = len(tables[0]) if tables else 0
    slots, positions, starts, used = [], [], [0], 0
    for r, row in enumerate(tables):
        held, add = max(0, lens[r]), max(0, new[r])
        add = min(add, tokens - len(slots))
        for at in range(-(-held // page), min(width, -(-(held + add) // page))):
            row[at] = free[used] if used < len(free) else -1
            used += 1
        for p in range(held, held + add):
            pg = row[p // page] if p // page < width else -1
            slots.append(pg * page + p % page if pg >= 0 else -1)
            positions.append(p)
        starts.append(len(slots))
    pad = tokens - len(slots)
    return tables, slots + [-1] * pad, positions + [0] * pad, starts, [used]


def run_tables(lens, new, tables, free, page, tokens):
    from tattn import page_tables

    t = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in (lens, new, tables, free)]
    if not tables:
        t[2] = torch.zeros(0, 4, dtype=torch.int32, device=DEV)
    got = page_tables(t[0], t[1], t[2], t[3], page, tokens)
    return [t[2].tolist(), *(x.tolist() for x in got)]


def make(rng, r, longest, most, page, spare=0, short=0, width=None):
    lens = rng.integers(0, longest + 1, r).tolist()
    new = rng.integers(0, most + 1, r).tolist()
    width = width or (longest + most + page - 1) // page + 1
    order = rng.permutation(r * width * 2 + 8).tolist()
    tables = [[order.pop() if at < -(-held // page) else -1 for at in range(width)] for held in lens]
    need = sum(-(-(a + b) // page) - -(-a // page) for a, b in zip(lens, new))
    free = [order.pop() if order else 7 for _ in range(max(0, need - short))]
    return lens, new, tables, free, page, sum(new) + spare


@pytest.mark.parametrize("r,longest,most,page", [
    (1, 0, 1, 16), (1, 31, 1, 16), (3, 40, 0, 32), (7, 100, 33, 16), (256, 300, 1, 16), (255, 500, 40, 64),
    (1024, 50, 3, 16), (1025, 20, 5, 128), (2100, 9, 2, 16), (5, 3000, 2500, 1024), (2, 10, 5000, 16),
])
def test_page_tables_match_a_loop(r, longest, most, page):
    rng = np.random.default_rng(r * 7 + page)
    case = make(rng, r, longest, most, page, spare=int(rng.integers(0, 2000)))
    print("page_tables", r, longest, most, page, case[5], flush=True)
    assert run_tables(*case) == [list(x) for x in expected_tables(*case)]


@pytest.mark.parametrize("r,short,width,cut", [(9, 3, None, 0), (9, 1000, None, 0), (9, 0, 3, 0), (9, 0, None, 100), (1500, 40, None, 900)])
def test_page_tables_where_pages_rows_or_tokens_run_out(r, short, width, cut):
    """Tokens without a page have slot -1 and the count says how many pages were needed; tokens past the list are not placed."""
    rng = np.random.default_rng(r + short + cut)
    lens, new, tables, free, page, tokens = make(rng, r, 60, 30, 16, short=short)
    if width:
        tables = [row[:width] for row in tables]
    case = (lens, new, tables, free, page, max(0, tokens - cut))
    assert run_tables(*case) == [list(x) for x in expected_tables(*case)]


def test_page_tables_without_requests_tokens_or_with_negative_lengths():
    assert run_tables([], [], [], [1, 2], 16, 5) == [[], [-1] * 5, [0] * 5, [0], [0]]
    case = ([5, 0], [0, 0], [[3, -1], [-1, -1]], [], 16, 0)
    assert run_tables(*case) == [list(x) for x in expected_tables(*case)]
    case = ([-4, 17], [3, -9], [[-1, -1], [2, 4]], [8, 9], 16, 6)
    assert run_tables(*case) == [list(x) for x in expected_tables(*case)]


def test_page_tables_in_a_slice_of_a_wider_table_and_in_a_graph():
    """Rows of a table with a stride of its own; captured, then replayed on new lengths."""
    from tattn import page_tables

    rng = np.random.default_rng(5)
    lens, new, tables, free, page, tokens = make(rng, 33, 90, 20, 16, spare=9)
    wide = torch.full((33, len(tables[0]) + 5), 99, dtype=torch.int32, device=DEV)
    tab = wide[:, 2:2 + len(tables[0])]
    t = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in (lens, new, free)]
    page_tables(t[0], t[1], tab.copy_(torch.tensor(tables)), t[2], page, tokens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = page_tables(t[0], t[1], tab, t[2], page, tokens)
    for seed in range(3):
        rng = np.random.default_rng(100 + seed)
        new = rng.integers(0, 21, 33).tolist()
        t[1].copy_(torch.tensor(new))
        tab.copy_(torch.tensor(tables))
        graph.replay()
        torch.cuda.synchronize()
        want = expected_tables(lens, new, tables, free, page, tokens)
        assert [tab.tolist(), *(x.tolist() for x in out)] == [list(x) for x in want]
        assert (wide[:, :2] == 99).all() and (wide[:, -3:] == 99).all()


# ---- the cache in 4 bits ------------------------------------------------------------------------

def held(x, dtype):
    """The definition on float64 values [.., d]: blocks of 32, smallest power of two with amax < 7 * 2^e (6 * 2^e
    finite in the type), nearest level, ties to the even mantissa (0, 1, 2, 4)."""
    most = int(np.floor(np.log2(torch.finfo(dtype).max / 6)))
    b = x.reshape(*x.shape[:-1], -1, 32)
    with np.errstate(invalid="ignore", divide="ignore"):
        top = np.abs(b).max(-1, keepdims=True)
        finite, none = np.isfinite(top), top < 2.0 ** -120
        e = np.floor(np.log2(np.where(finite & ~none, top, 1.0))) - 2
        e = np.minimum(e + (top >= 7 * 2.0 ** e), most)
        y = np.abs(b) / 2.0 ** e
        gap = np.abs(y[..., None] - LEVELS)
        tied = gap == gap.min(-1, keepdims=True)
        at = (tied * (1 + (np.arange(8) % 2 == 0))).argmax(-1)
        out = np.where(none, 0.0, np.where(finite, np.copysign(LEVELS[at], b) * 2.0 ** e, np.nan))
    return out.reshape(x.shape)


def same(got, want):
    return np.array_equal(got, want, equal_nan=True)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("tokens,heads,page", [(1, 1, 16), (17, 3, 16), (100, 2, 64), (33, 8, 1024)])
def test_write_then_read_gives_the_held_values(dtype, d, tokens, heads, page):
    from tattn import Cache4, cache4_read, cache4_write

    g = torch.Generator().manual_seed(tokens * d + page)
    kv = torch.randn(tokens, 2, heads, d, generator=g) * torch.exp2(torch.randint(-9, 9, (tokens, 2, heads, 1), generator=g))
    kv = kv.to(dtype)
    pages = (tokens + page - 1) // page + 2
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    slots[tokens // 2] = (-1, pages * page, 1 << 40)[tokens % 3] if tokens > 1 else slots[0]
    cache = Cache4.empty(pages, page, heads, d, dtype=dtype, device=DEV)
    cache.codes.fill_(0x11)
    before = cache.codes.clone()
    dev = kv.to(DEV)
    print("cache4", dtype, d, tokens, heads, page, flush=True)
    cache4_write(cache, dev[:, 0], dev[:, 1], slots.to(DEV))
    k, v = cache4_read(cache, slots.to(DEV))
    want = held(kv.double().numpy(), dtype)
    want[[s < 0 or s >= pages * page for s in slots.tolist()]] = 0
    assert k.dtype == v.dtype == dtype and k.shape == (tokens, heads, d)
    assert same(k.double().cpu().numpy(), want[:, 0]) and same(v.double().cpu().numpy(), want[:, 1])
    # Nothing but the slots was touched.
    free = torch.ones(pages * page, dtype=torch.bool)
    free[[s for s in slots.tolist() if 0 <= s < pages * page]] = False
    flat = lambda c: c.permute(0, 3, 1, 2, 4).reshape(pages * page, -1)
    assert torch.equal(flat(cache.codes)[free.to(DEV)], flat(before)[free.to(DEV)])
    # The layout that the class documents, decoded by hand.
    real = [i for i, s in enumerate(slots.tolist()) if 0 <= s < pages * page]
    at = slots[real]
    c = cache.codes.cpu()[at // page, :, :, at % page].numpy()
    e = cache.scales.cpu()[at // page, :, :, at % page].double().numpy()
    x = np.stack((c & 15, c >> 4), -1).reshape(*c.shape[:-1], d)
    x = np.where(x < 8, 1, -1) * LEVELS[x & 7]
    x = x * np.repeat(2.0 ** (e - 127), 32, -1)
    assert same(x[:, :, 0], want[real, 0]) and same(x[:, :, 1], want[real, 1])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_every_16_bit_value_alone_and_beside_a_larger_one(dtype):
    """Each finite magnitude as the only value of a block, and beside block maxima of 4, 5, 6, 7 and 15/2 (in both
    types the borders between levels and the step in the scale are hit exactly)."""
    from tattn import Cache4, cache4_read, cache4_write

    bits = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(dtype)
    rows = torch.zeros(1 << 16, 32, dtype=dtype)
    rows[:, 5] = bits
    cache = Cache4.empty((1 << 16) // 1024, 1024, 1, 32, dtype=dtype, device=DEV)
    slots = torch.arange(1 << 16, device=DEV)
    for top in (0.0, 4.0, 5.0, 6.0, 7.0, 7.5):
        rows[:, 9] = top
        x = rows.to(DEV)[:, None]
        cache4_write(cache, x, x.flip(0), slots)
        k, v = cache4_read(cache, slots)
        want = held(rows.double().numpy(), dtype)
        assert same(k.double().cpu().numpy()[:, 0], want)
        assert same(v.double().cpu().numpy()[:, 0], want[::-1])


def test_strided_rows_copies_and_graphs():
    """k and v as slices of one projection, an odd offset that is copied, and a captured write and read."""
    from tattn import Cache4, cache4_read, cache4_write

    g = torch.Generator().manual_seed(3)
    qkv = torch.randn(40, 12, 64, generator=g).half().to(DEV)
    k, v = qkv[:, 8:10], qkv[:, 10:]
    slots = torch.arange(40, device=DEV) + 3
    cache = Cache4.empty(4, 16, 2, 64, dtype=torch.float16, device=DEV)
    cache4_write(cache, k, v, slots)
    want = [held(t.double().cpu().numpy(), torch.float16) for t in (k, v)]
    for got, w in zip(cache4_read(cache, slots), want):
        assert same(got.double().cpu().numpy(), w)
    flat = torch.randn(40 * 128 + 1, generator=g).half().to(DEV)
    odd = flat[1:].view(40, 2, 64)
    cache4_write(cache, odd, v, slots)
    assert same(cache4_read(cache, slots)[0].double().cpu().numpy(), held(odd.double().cpu().numpy(), torch.float16))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache4_write(cache, k, v, slots)
        out = cache4_read(cache, slots)
    for seed in range(3):
        qkv.copy_(torch.randn(40, 12, 64, generator=g).half())
        cache.codes.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for got, t in zip(out, (k, v)):
            assert same(got.double().cpu().numpy(), held(t.double().cpu().numpy(), torch.float16))


def test_no_tokens():
    from tattn import Cache4, cache4_read, cache4_write

    cache = Cache4.empty(2, 16, 2, 64, dtype=torch.float16, device=DEV)
    none = torch.zeros(0, 2, 64, dtype=torch.float16, device=DEV)
    at = torch.zeros(0, dtype=torch.int64, device=DEV)
    cache4_write(cache, none, none, at)
    assert cache4_read(cache, at)[0].shape == (0, 2, 64)
    assert not cache.codes.any()
