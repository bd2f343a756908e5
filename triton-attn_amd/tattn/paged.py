"""A paged key/value cache held in 4 bits, and the page bookkeeping of a serving step.

    tables, slots, ... = page_tables(...)     # pages and slots of the tokens that requests add
    cache4_write(cache, k, v, slots)          # their keys and values into the cache
    cache4_read(cache, slots)                 # what the cache holds for them
    cache4_attention(q, cache, tables, lens)  # one token per request over its pages

No counterpart in the reference. Lengths, tables and slots stay on the GPU: no call waits for it, and
every call can be captured into a graph. Values the GPU alone knows are checked there: a slot or page outside
the cache is skipped, as documented per call.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from tattn import _lib
from tattn._args import aligned, check_index, layouts, no_tangents, remember, rows_apart, same_device, strides, whole
from tattn.api import _on_device, _require_gpu, _stream

_DTYPES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}

PAGE_SIZES = (16, 32, 64, 128, 256, 512, 1024)


def _check_page_size(page_size: int) -> None:
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page size must be a power of two from 16 to 1024, got {page_size}")


class PageTables(NamedTuple):
    slots: torch.Tensor      # int64 [tokens]: page * page_size + offset; -1 without a page
    positions: torch.Tensor  # int32 [tokens]: position within the request
    starts: torch.Tensor     # int32 [requests + 1]: where each request's tokens begin
    taken: torch.Tensor      # int32 [1]: pages needed from the free list


_table_plans: dict[tuple, tuple] = {}


def _check_tables(lens, new_tokens, tables, free_pages, page_size) -> None:
    if lens.dim() != 1 or lens.dtype != torch.int32:
        raise ValueError(f"lens must be int32 [requests], got {lens.dtype} {list(lens.shape)}")
    r = lens.shape[0]
    check_index("new_tokens", new_tokens, torch.int32, (r,))
    if tables.dim() != 2:
        raise ValueError(f"tables must be int32 [requests, width], got {list(tables.shape)}")
    check_index("tables", tables, torch.int32, (r, tables.shape[1]))
    if free_pages.dim() != 1 or free_pages.dtype != torch.int32:
        raise ValueError(f"free_pages must be int32 [pages], got {free_pages.dtype} {list(free_pages.shape)}")
    if tables.numel() and ((tables.shape[1] > 1 and tables.stride(1) != 1) or (r > 1 and tables.stride(0) < tables.shape[1])):
        raise ValueError("tables is updated in place: its rows must be contiguous and must not overlap")
    _check_page_size(page_size)
    same_device(lens, new_tokens=new_tokens, tables=tables, free_pages=free_pages)


def page_tables(lens: torch.Tensor, new_tokens: torch.Tensor, tables: torch.Tensor, free_pages: torch.Tensor,
                page_size: int, tokens: int) -> PageTables:
    """Pages and slots for the tokens that requests add to a paged cache, on the GPU.

    lens, new_tokens: int32 [requests], tokens held and added. tables: int32 [requests, width], the pages
    of each request, extended in place with pages from free_pages (int32 [any]) in request order. tokens: length of the
    returned lists, the batch's padded token count; entries behind the last request have slot -1 and position 0, and
    tokens past it are not placed (no slot, no page). lens and free_pages are not changed: the caller adds new_tokens
    and skips `taken` pages. Where free pages or a table row run out, tokens have slot -1 (and `taken` exceeds the list).
    """
    page_size, tokens = whole("page_size", page_size), whole("tokens", tokens)
    if not 0 <= tokens < (1 << 31) - 4096:
        raise ValueError(f"tokens out of range: {tokens}")
    key = (layouts(lens, new_tokens, tables, free_pages), page_size)
    plan = _table_plans.get(key)
    if plan is None:
        _check_tables(lens, new_tokens, tables, free_pages, page_size)
        _require_gpu(lens)
        plan = remember(_table_plans, key, (*tables.shape, tables.stride(0), free_pages.shape[0]))
    r, width, row, pages = plan
    lens, new_tokens, free_pages = lens.contiguous(), new_tokens.contiguous(), free_pages.contiguous()
    slots = lens.new_empty(tokens, dtype=torch.int64)
    positions, starts, taken = lens.new_empty(tokens), lens.new_empty(r + 1), lens.new_empty(1)
    with _on_device(lens):
        rc = _lib.load().tattn_page_tables(
            lens.data_ptr(), new_tokens.data_ptr(), tables.data_ptr(), free_pages.data_ptr(), slots.data_ptr(),
            positions.data_ptr(), starts.data_ptr(), taken.data_ptr(), r, width, row, pages, tokens, page_size, _stream(lens))
    if rc:
        _lib.check(rc, "tattn_page_tables")
    return PageTables(slots, positions, starts, taken)


class Cache4:
    """Keys and values of a paged cache in 4 bits (4.25 with their exponents).

    codes: uint8 [pages, kv_heads, 2, page_size, head_dim / 2] (2: keys, values; an even d in the low half of a
    byte), e2m1 codes (sign, two exponent bits, one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6). scales: uint8 [pages,
    kv_heads, 2, page_size, head_dim / 32], biased exponents of the blocks of 32 values along the head: the smallest power
    of two at which the block's largest magnitude rounds to 6 or less (and 6 times which is finite in dtype). A block that
    held an infinity or a NaN reads as NaN.
    dtype: float16 or bfloat16, the type of the values written and read, and of the queries over them.
    """

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype) -> None:
        if codes.dim() != 5 or codes.dtype != torch.uint8 or codes.shape[2] != 2:
            raise ValueError(f"codes must be uint8 [pages, kv_heads, 2, page_size, head_dim / 2], got {codes.dtype} {list(codes.shape)}")
        pages, heads, _, page, half = codes.shape
        if 2 * half not in (32, 64, 128):
            raise ValueError(f"head dim must be 32, 64 or 128, got {2 * half}")
        if heads < 1:
            raise ValueError("expected at least one kv head")
        check_index("scales", scales, torch.uint8, (pages, heads, 2, page, half // 16))
        _check_page_size(page)
        if dtype not in _DTYPES:
            raise ValueError(f"dtype must be float16 or bfloat16, got {dtype}")
        same_device(codes, scales=scales)
        if not (codes.is_contiguous() and scales.is_contiguous()) or codes.data_ptr() % 16 or scales.data_ptr() % 4:
            raise ValueError("codes and scales must be contiguous, codes 16-byte and scales 4-byte aligned")
        self.codes, self.scales, self.dtype = codes, scales, dtype
        self.pages, self.kv_heads, self.page_size, self.head_dim = pages, heads, page, 2 * half
        self.layout = (codes.shape, dtype, codes.device)
        self.sizes = (heads, 2 * half, pages, page, _DTYPES[dtype])

    @classmethod
    def empty(cls, pages: int, page_size: int, kv_heads: int, head_dim: int, *, dtype: torch.dtype,
              device: torch.device | str) -> "Cache4":
        """A cache of zeros."""
        shape = (pages, kv_heads, 2, page_size)
        return cls(torch.zeros((*shape, head_dim // 2), dtype=torch.uint8, device=device),
                   torch.zeros((*shape, head_dim // 32), dtype=torch.uint8, device=device), dtype)


_write_plans: dict[tuple, tuple] = {}


def cache4_write(cache: Cache4, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Writes keys and values [tokens, kv_heads, head_dim] (the cache's dtype, any token and head strides) into
    `slots` (int64 [tokens], as page_tables gives them). Slots outside the cache, such as a padded token's -1,
    are skipped. No two tokens of a call may share a slot. Gradients do not flow through the cache; forward-mode derivatives
    are refused."""
    no_tangents(k, v)
    key = (layouts(k, v, slots), cache.layout)
    plan = _write_plans.get(key)
    if plan is None:
        if k.dim() != 3 or k.shape != v.shape or tuple(k.shape[1:]) != (cache.kv_heads, cache.head_dim):
            raise ValueError(f"expected k, v of shape [tokens, {cache.kv_heads}, {cache.head_dim}]; got {list(k.shape)}, {list(v.shape)}")
        if k.dtype != cache.dtype or v.dtype != cache.dtype:
            raise ValueError(f"k and v must have the cache's dtype {cache.dtype}, got {k.dtype}, {v.dtype}")
        check_index("slots", slots, torch.int64, (k.shape[0],))
        same_device(cache.codes, k=k, v=v, slots=slots)
        _require_gpu(k)
        plan = remember(_write_plans, key, (rows_apart(k), rows_apart(v), strides(k, v)))
    given = k, v
    k, v, slots = aligned(k, plan[0]), aligned(v, plan[1]), slots.contiguous()
    _, st = plan[2] if k is given[0] and v is given[1] else strides(k, v)
    with _on_device(k):
        rc = _lib.load().tattn_cache4_write(
            cache.codes.data_ptr(), cache.scales.data_ptr(), k.data_ptr(), v.data_ptr(), slots.data_ptr(), *st, k.shape[0],
            *cache.sizes, _stream(k))
    if rc:
        _lib.check(rc, "tattn_cache4_write")


def cache4_read(cache: Cache4, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(K, V) [tokens, kv_heads, head_dim]: the values the cache holds for `slots` (int64 [tokens]); zeros for slots
    outside it. For prompts that continue a cached prefix, and to see what 4 bits made of a tensor."""
    if slots.dim() != 1 or slots.dtype != torch.int64:
        raise ValueError(f"slots must be int64 [tokens], got {slots.dtype} {list(slots.shape)}")
    if slots.device != cache.codes.device:
        same_device(cache.codes, slots=slots)
    _require_gpu(slots)
    slots = slots.contiguous()
    n = slots.shape[0]
    shape = (n, cache.kv_heads, cache.head_dim)
    k, v = slots.new_empty(shape, dtype=cache.dtype), slots.new_empty(shape, dtype=cache.dtype)
    with _on_device(slots):
        rc = _lib.load().tattn_cache4_read(cache.codes.data_ptr(), cache.scales.data_ptr(), k.data_ptr(), v.data_ptr(),
                                           slots.data_ptr(), n, *cache.sizes, _stream(slots))
    if rc:
        _lib.check(rc, "tattn_cache4_read")
    return k, v


_attention_plans: dict[tuple, tuple] = {}


def _attention_plan(q, cache, tables, lens, window, sinks) -> tuple:
    """Checks a call of cache4_attention; whether q and tables are copied, the strides of q and the output (None where q is
    copied), the float32 values of workspace, and the sizes among the launch's arguments (None: nothing to see)."""
    if q.dim() != 3 or q.shape[2] != cache.head_dim or q.shape[1] < 1 or q.shape[1] % cache.kv_heads:
        raise ValueError(f"expected q [requests, heads, {cache.head_dim}] with a multiple of {cache.kv_heads} heads; got {list(q.shape)}")
    r, h, d = q.shape
    if q.dtype != cache.dtype:
        raise ValueError(f"q must have the cache's dtype {cache.dtype}, got {q.dtype}")
    if tables.dim() != 2:
        raise ValueError(f"tables must be int32 [requests, width], got {list(tables.shape)}")
    width = tables.shape[1]
    check_index("tables", tables, torch.int32, (r, width))
    check_index("lens", lens, torch.int32, (r,))
    if (window is not None and window < 1) or sinks < 0:
        raise ValueError(f"window must be positive and sinks not negative, got {window} and {sinks}")
    same_device(q, cache=cache.codes, tables=tables, lens=lens)
    _require_gpu(q)
    if q.numel() == 0 or width == 0 or cache.pages == 0:
        return rows_apart(q), False, None, 0, None
    held = width * cache.page_size
    window, sinks = 0 if window is None else min(window, held), min(sinks, held)
    out = ctypes.c_int64()
    _lib.check(_lib.load().tattn_cache4_attention_workspace(r, h, cache.kv_heads, d, width, cache.page_size, window, sinks,
                                                            ctypes.byref(out)), "tattn_cache4_attention_workspace")
    return (rows_apart(q), width > 1 and tables.stride(1) != 1,
            None if rows_apart(q) else strides(q, torch.empty_like(q)), out.value,
            (r, h, cache.kv_heads, d, width, cache.pages, cache.page_size, window, sinks, _DTYPES[cache.dtype]))


def cache4_attention(
    q: torch.Tensor, cache: Cache4, tables: torch.Tensor, lens: torch.Tensor, window: int | None = None, sinks: int = 0,
    sm_scale: float | None = None,
) -> torch.Tensor:
    """Attention of one token per request over the cache: q [requests, heads, head_dim] (the cache's dtype; heads a
    multiple of its kv heads, consecutive heads sharing one; any request and head strides), tables int32 [requests, width]
    as page_tables keeps them, lens int32 [requests]: tokens each request sees, the newest one included (clamped to what its
    table row holds). With a window only the last `window` tokens and the first `sinks` are seen, and pages without a seen
    token are not looked up (they may have been given away). Tokens on a page number outside the cache are hidden; a request
    that sees nothing gives zeros. sm_scale defaults to 1 / sqrt(head_dim). For serving: refuses a q that requires gradients or
    carries forward-mode ones."""
    no_tangents(q)
    if q.requires_grad and torch.is_grad_enabled():
        raise ValueError("cache4_attention has no gradients: call it under torch.no_grad()")
    window, sinks = None if window is None else whole("window", window), whole("sinks", sinks)
    key = (layouts(q, tables, lens), cache.layout, window, sinks)
    plan = _attention_plans.get(key)
    if plan is None:
        plan = remember(_attention_plans, key, _attention_plan(q, cache, tables, lens, window, sinks))
    copy_q, copy_tables, held, floats, sizes = plan
    given = q
    q, lens = aligned(q, copy_q), lens.contiguous()
    o = torch.empty_like(q)
    if sizes is None:
        return o.zero_()
    if copy_tables:
        tables = tables.contiguous()
    work = q.new_empty(floats, dtype=torch.float32) if floats else None
    _, st = held if held and q is given else strides(q, o)
    with _on_device(q):
        rc = _lib.load().tattn_cache4_attention(
            q.data_ptr(), o.data_ptr(), cache.codes.data_ptr(), cache.scales.data_ptr(), tables.data_ptr(), lens.data_ptr(),
            None if work is None else work.data_ptr(), *st, tables.stride(0), *sizes,
            float(sm_scale) if sm_scale is not None else cache.head_dim ** -0.5, _stream(q))
    if rc:
        _lib.check(rc, "tattn_cache4_attention")
    return o
