"""Attention over a sliding window and the first keys, for training, prompts and single tokens.

    o = window_attention(q, k, v, window=1024, sinks=4)             # training, or a prompt
    o = window_attention(q, k_cache, v_cache, 1024, 4, lens=lens)    # the newest tokens over a 16-bit cache

No counterpart in the reference, whose attention is causal over all keys or unmasked.
"""

from __future__ import annotations

import ctypes
import math
from typing import Any

import torch
from torch.autograd.function import once_differentiable

from tattn import _lib
from tattn._args import aligned, check_index, layouts, no_tangents, remember, rows_apart, same_device, strides, whole
from tattn.api import _DTYPES, _on_device, _require_gpu, _stream


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
        raise ValueError(f"q, k, v must share dtype float16, bfloat16 or float32, got {q.dtype}, {k.dtype}, {v.dtype}")
    if window < 1 or sinks < 0:
        raise ValueError(f"window must be positive and sinks not negative, got {window} and {sinks}")
    same_device(q, k=k, v=v, lens=lens)
    if lens is not None:
        check_index("lens", lens, torch.int32, (z,))
    elif n > s:
        raise ValueError(f"{n} queries for {s} keys: the queries are the last of the keys' positions")


def _tiles_apart(t: torch.Tensor) -> bool:
    """Whether the kernels cannot read t in tiles of rows where it lies: aligned rows that do not overlap, heads within
    31-bit offsets."""
    n, st, d = t.shape[2], t.stride(2), t.shape[3]
    return rows_apart(t) or (n > 1 and (st < d or st > 1 << 24 or (n + 256) * st * t.element_size() >= 0x7FFFFF00))


def _tiles(t: torch.Tensor) -> torch.Tensor:
    return aligned(t, _tiles_apart(t))


def _workspace(backward: bool, sizes: tuple) -> int:
    """Float32 values of workspace that a call of these sizes needs."""
    out = ctypes.c_int64()
    _lib.check(_lib.load().tattn_window_workspace(int(backward), *sizes, ctypes.byref(out)), "tattn_window_workspace")
    return out.value


_plans: dict[tuple, tuple] = {}


def _plan(q, k, v, window, sinks, lens) -> tuple:
    """Checks a call; which of q, k, v are copied, the strides of inputs and output (None where one is copied), the float32
    values of workspace of forward and backward and of delta, and the sizes among the launches' arguments (None: nothing to see)."""
    _check(q, k, v, window, sinks, lens)
    _require_gpu(q)
    copies = tuple(_tiles_apart(t) for t in (q, k, v))
    z, h, n, d = q.shape
    hk, s = k.shape[1:3]
    if q.numel() == 0 or s == 0:
        return copies, None, 0, 0, 0, None
    sizes = (z, h, hk, n, s, d, min(window, s), min(sinks, s))
    half = q.dtype != torch.float32  # float32 is never split
    norms = 1 + 2 * z * hk * ((n * (h // hk) + 127) // 128) if q.dtype == torch.float16 else 0
    return (copies, None if any(copies) else strides(q, k, v, torch.empty_like(q)), _workspace(False, sizes) if half else 0,
            _workspace(True, sizes) if half and lens is None else 0, z * h * n + norms, (*sizes, _DTYPES[q.dtype]))


def _forward(q, k, v, plan, scale, lens, save_lse) -> tuple[torch.Tensor, torch.Tensor | None]:
    copies, held, floats, _, _, sizes = plan
    given = q, k, v
    q, k, v = aligned(q, copies[0]), aligned(k, copies[1]), aligned(v, copies[2])
    o = torch.empty_like(q)
    m = q.new_empty(q.shape[:3], dtype=torch.float32) if save_lse else None
    if sizes is None:
        return o.zero_(), m
    work = q.new_empty(floats, dtype=torch.float32) if floats else None
    _, st = held if held and q is given[0] and k is given[1] and v is given[2] else strides(q, k, v, o)
    with _on_device(q):
        rc = _lib.load().tattn_window_fwd(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), None if m is None else m.data_ptr(),
            None if lens is None else lens.data_ptr(), None if work is None else work.data_ptr(), *st, *sizes, scale, _stream(q))
    if rc:
        _lib.check(rc, "tattn_window_fwd")
    return o, m


def _backward(q, k, v, o, m, do, plan, scale) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    floats, rows, sizes = plan[3:]
    q, k, v, o, do = _tiles(q), _tiles(k), _tiles(v), _tiles(o), _tiles(do)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    if sizes is None:
        return dq.zero_(), dk.zero_(), dv.zero_()
    delta = m.new_empty(rows)
    work = q.new_empty(floats, dtype=torch.float32) if floats else None
    _, st = strides(q, k, v, o, do, dq, dk, dv)
    with _on_device(q):
        rc = _lib.load().tattn_window_bwd(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), do.data_ptr(), dq.data_ptr(), dk.data_ptr(),
            dv.data_ptr(), m.data_ptr(), delta.data_ptr(), None if work is None else work.data_ptr(), *st, *sizes, scale,
            _stream(q))
    if rc:
        _lib.check(rc, "tattn_window_bwd")
    return dq, dk, dv


class _Window(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, q, k, v, plan, scale):
        o, m = _forward(q, k, v, plan, scale, None, True)
        ctx.save_for_backward(q, k, v, o, m)
        ctx.args = plan, scale
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, do):
        return (*_backward(*ctx.saved_tensors, do, *ctx.args), None, None)


def window_attention(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int, sinks: int = 0, sm_scale: float | None = None,
    lens: torch.Tensor | None = None,
) -> torch.Tensor:
    """Causal attention in which a query sees the last `window` keys, its own included, and the first `sinks` keys.

    q [batch, heads, queries, dim]; k, v [batch, kv heads, keys, dim]; float16, bfloat16 or float32; heads a multiple of
    kv heads, consecutive heads sharing one; any strides. The queries are the last ones of the keys' positions: query n of
    a sequence with len keys is at position len - queries + n and sees key j <= position with position - j < window or
    j < sinks. len is keys, or lens[batch] (int32, on the GPU, clamped to [0, keys]) where a cache is filled to
    different lengths; what lies behind it, or before every window, reaches no result. Rows at positions below 0 give
    zeros. sm_scale defaults to 1 / sqrt(dim). Differentiable in q, k and v without lens; with lens the call is for serving
    and refuses inputs that require gradients. Forward-mode derivatives are refused. A key or value that is infinite or NaN
    makes the rows that see it NaN, and may make NaN of rows up to 64 positions before it or after its window that do not see
    it."""
    no_tangents(q, k, v)
    window, sinks = whole("window", window), whole("sinks", sinks)
    key = (layouts(q, k, v, lens), window, sinks)
    plan = _plans.get(key)
    needs = (q.requires_grad or k.requires_grad or v.requires_grad) and torch.is_grad_enabled()
    if needs and lens is not None:
        raise ValueError("no gradients with lens: call it under torch.no_grad(), or without lens")
    if plan is None:
        plan = remember(_plans, key, _plan(q, k, v, window, sinks, lens))
    scale = float(sm_scale) if sm_scale is not None else 1.0 / math.sqrt(q.shape[3])
    if needs:
        return _Window.apply(q, k, v, plan, scale)
    return _forward(q, k, v, plan, scale, None if lens is None else lens.contiguous(), False)[0]
