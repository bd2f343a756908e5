"""Attention over a sliding window and the first keys, for training, prompts and single tokens.

    o = window_attention(q, k, v, window=1024, sinks=4)             # training, or a prompt
    o = window_attention(q, k_cache, v_cache, 1024, 4, lens=lens)    # the newest tokens over a 16-bit cache

No counterpart in the reference, whose attention is causal over all keys or unmasked.
"""

from __future__ import annotations

import ctypes
import functools
import math
from typing import Any

import torch
from torch.autograd.function import once_differentiable

from tattn import _lib
from tattn._args import check_index, rows, same_device, strides
from tattn.api import _on_device, _require_gpu, _stream

_DTYPES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


def _check(q, k, v, window, sinks, lens) -> None:
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise ValueError(f"expected q [batch, heads, queries, dim] and k, v of equal shape [batch, kv heads, keys, dim]; "
                         f"got {q.shape}, {k.shape}, {v.shape}")
    z, h, n, d = q.shape
    hk, s = k.shape[1:3]
    if d not in (16, 32, 64, 128):
        raise ValueError(f"head dim must be 16, 32, 64 or 128, got {d}")
    if hk < 1 or h < 1 or h % hk:
        raise ValueError(f"heads must be a multiple of kv heads, got {h} and {hk}")
    if not (q.dtype == k.dtype == v.dtype) or q.dtype not in _DTYPES:
        raise ValueError(f"q, k, v must share dtype float16 or bfloat16, got {q.dtype}, {k.dtype}, {v.dtype}")
    if window < 1 or sinks < 0:
        raise ValueError(f"window must be positive and sinks not negative, got {window} and {sinks}")
    same_device(q, k=k, v=v, lens=lens)
    if lens is not None:
        check_index("lens", lens, torch.int32, (z,))
    elif n > s:
        raise ValueError(f"{n} queries for {s} keys: the queries are the last of the keys' positions")


def _tiles(t: torch.Tensor) -> torch.Tensor:
    """t itself where the kernels read its rows in tiles (aligned rows that do not overlap, heads within 31-bit
    offsets), else an aligned contiguous copy."""
    t = rows(t)
    n, st, d = t.shape[2], t.stride(2), t.shape[3]
    if n > 1 and (st < d or st > 1 << 24 or (n + 256) * st * 2 >= 0x7FFFFF00):
        t = t.clone(memory_format=torch.contiguous_format)
    return t


@functools.lru_cache(maxsize=4096)
def _workspace(backward: bool, z: int, h: int, hk: int, n: int, s: int, d: int, window: int, sinks: int) -> int:
    """Float32 values of workspace that a call of these sizes needs."""
    out = ctypes.c_int64()
    _lib.check(_lib.load().tattn_window_workspace(int(backward), z, h, hk, n, s, d, window, sinks, ctypes.byref(out)),
               "tattn_window_workspace")
    return out.value


def _sizes(q, k, window, sinks) -> tuple:
    z, h, n, d = q.shape
    hk, s = k.shape[1:3]
    return z, h, hk, n, s, d, min(window, s), min(sinks, s)


def _forward(q, k, v, window, sinks, scale, lens, save_lse) -> tuple[torch.Tensor, torch.Tensor | None]:
    q, k, v = _tiles(q), _tiles(k), _tiles(v)
    o = torch.empty_like(q)
    m = q.new_empty(q.shape[:3], dtype=torch.float32) if save_lse else None
    if q.numel() == 0 or k.shape[2] == 0:
        return o.zero_(), m
    sizes = _sizes(q, k, window, sinks)
    n = _workspace(False, *sizes)
    work = q.new_empty(n, dtype=torch.float32) if n else None
    _, st = strides(q, k, v, o)
    with _on_device(q):
        rc = _lib.load().tattn_window_fwd(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), None if m is None else m.data_ptr(),
            None if lens is None else lens.data_ptr(), None if work is None else work.data_ptr(), *st, *sizes,
            _DTYPES[q.dtype], scale, _stream(q))
    _lib.check(rc, "tattn_window_fwd")
    return o, m


def _backward(q, k, v, o, m, do, window, sinks, scale) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    q, k, v, o, do = _tiles(q), _tiles(k), _tiles(v), _tiles(o), _tiles(do)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    if q.numel() == 0 or k.numel() == 0:
        return dq.zero_(), dk.zero_(), dv.zero_()
    delta = torch.empty_like(m)
    sizes = _sizes(q, k, window, sinks)
    n = _workspace(True, *sizes)
    work = q.new_empty(n, dtype=torch.float32) if n else None
    _, st = strides(q, k, v, o, do, dq, dk, dv)
    with _on_device(q):
        rc = _lib.load().tattn_window_bwd(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), do.data_ptr(), dq.data_ptr(), dk.data_ptr(),
            dv.data_ptr(), m.data_ptr(), delta.data_ptr(), None if work is None else work.data_ptr(), *st, *sizes,
            _DTYPES[q.dtype], scale, _stream(q))
    _lib.check(rc, "tattn_window_bwd")
    return dq, dk, dv


class _Window(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, q, k, v, window, sinks, scale):
        o, m = _forward(q, k, v, window, sinks, scale, None, True)
        ctx.save_for_backward(q, k, v, o, m)
        ctx.args = window, sinks, scale
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, do):
        return (*_backward(*ctx.saved_tensors, do, *ctx.args), None, None, None)


def window_attention(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int, sinks: int = 0, sm_scale: float | None = None,
    lens: torch.Tensor | None = None,
) -> torch.Tensor:
    """Causal attention in which a query sees the last `window` keys, its own included, and the first `sinks` keys.

    q [batch, heads, queries, dim]; k, v [batch, kv heads, keys, dim]; float16 or bfloat16; heads a multiple of kv heads,
    consecutive heads sharing one; any strides. The queries are the last ones of the keys' positions: query n of a
    sequence with len keys is at position len - queries + n and sees key j <= position with position - j < window or
    j < sinks. len is keys, or lens[batch] (int32, on the GPU, clamped to [0, keys]) where a cache is filled to
    different lengths; what lies behind it, or before every window, reaches no result. Rows at positions below 0 give
    zeros. sm_scale defaults to 1 / sqrt(dim). Differentiable in q, k and v without lens; with lens the call is for serving
    and refuses inputs that require gradients. A key or value that is infinite or NaN makes the rows that see it
    NaN, and may make NaN of rows up to 64 positions before it or after its window that do not see it."""
    _check(q, k, v, window, sinks, lens)
    needs = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    if needs and lens is not None:
        raise ValueError("no gradients with lens: call it under torch.no_grad(), or without lens")
    _require_gpu(q)
    scale = float(sm_scale) if sm_scale is not None else 1.0 / math.sqrt(q.shape[3])
    if lens is not None:
        lens = lens.contiguous()
    if needs:
        return _Window.apply(q, k, v, int(window), int(sinks), scale)
    return _forward(q, k, v, int(window), int(sinks), scale, lens, False)[0]
