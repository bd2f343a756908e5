"""Attention over keys of another length: an encoder's states, and a prefix that a batch shares.

    o = cross_attention(q, k, v, lens=states)                    # training, passages, and one token
    o = prefix_attention(q, prefix_k, prefix_v, k, v, lens)      # the newest tokens of sequences behind one prefix

No counterpart in the reference, whose queries and keys are of one length and one sequence.
"""

from __future__ import annotations

import ctypes
import math
from typing import Any

import torch
from torch.autograd.function import once_differentiable

from tattn import _lib
from tattn._args import aligned, check_index, layouts, no_tangents, remember, rows_apart, same_device, strides
from tattn.api import _DTYPES, _on_device, _require_gpu, _stream
from tattn.window import _tiles_apart


def _check_heads(q, k, v, names: str) -> None:
    """Dimensions, head dim, heads and types, for queries and the keys and values `names`."""
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or q.shape[3] != k.shape[3]:
        raise ValueError(f"expected q [batch, heads, queries, dim] and {names} of equal shape [batch, kv heads, keys, dim]; "
                         f"got {q.shape}, {k.shape}, {v.shape}")
    if q.shape[3] not in (16, 32, 64, 128):
        raise ValueError(f"head dim must be 16, 32, 64 or 128, got {q.shape[3]}")
    if k.shape[1] < 1 or q.shape[1] < 1 or q.shape[1] % k.shape[1]:
        raise ValueError(f"heads must be a multiple of kv heads, got {q.shape[1]} and {k.shape[1]}")


def _check_cross(q, k, v, lens) -> None:
    _check_heads(q, k, v, "k, v")
    if q.shape[0] != k.shape[0]:
        raise ValueError(f"q, k, v must share their batch, got {q.shape[0]} and {k.shape[0]}")
    if not (q.dtype == k.dtype == v.dtype) or q.dtype not in _DTYPES:
        raise ValueError(f"q, k, v must share dtype float16, bfloat16 or float32, got {q.dtype}, {k.dtype}, {v.dtype}")
    same_device(q, k=k, v=v, lens=lens)
    if lens is not None:
        check_index("lens", lens, torch.int32, (q.shape[0],))


def _workspace(backward: bool, sizes: tuple) -> int:
    """Float32 values of workspace that a call of these sizes needs."""
    out = ctypes.c_int64()
    _lib.check(_lib.load().tattn_cross_workspace(int(backward), *sizes, ctypes.byref(out)), "tattn_cross_workspace")
    return out.value


_plans: dict[tuple, tuple] = {}


def _plan(q, k, v, lens) -> tuple:
    """Checks a call; which of q, k, v are copied, the strides of inputs and output (None where one is copied), the float32
    values of workspace of forward and backward, the sizes among the launches' arguments (None: nothing to see), and what the
    backward found for its five inputs in each layout: which are copied, and all strides."""
    _check_cross(q, k, v, lens)
    _require_gpu(q)
    copies = rows_apart(q), _tiles_apart(k), _tiles_apart(v)
    z, h, n, d = q.shape
    hk, s = k.shape[1:3]
    if q.numel() == 0 or s == 0:
        return copies, None, 0, 0, None, {}
    sizes = (z, h, hk, n, s, d, _DTYPES[q.dtype])
    return (copies, None if any(copies) else strides(q, k, v, torch.empty_like(q)), _workspace(False, sizes),
            _workspace(True, sizes), sizes, {})


def _forward(q, k, v, lens, plan, scale, save_lse) -> tuple[torch.Tensor, torch.Tensor | None]:
    copies, held, floats, _, sizes, _ = plan
    given = q, k, v
    q, k, v = aligned(q, copies[0]), aligned(k, copies[1]), aligned(v, copies[2])
    o = torch.empty_like(q)
    m = q.new_empty(q.shape[:3], dtype=torch.float32) if save_lse else None
    if sizes is None:
        return o.zero_(), m
    work = q.new_empty(floats, dtype=torch.float32) if floats else None
    _, st = held if held and q is given[0] and k is given[1] and v is given[2] else strides(q, k, v, o)
    with _on_device(q):
        rc = _lib.load().tattn_cross_fwd(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), None if m is None else m.data_ptr(),
            None if lens is None else lens.data_ptr(), None if work is None else work.data_ptr(), *st, *sizes, scale, _stream(q))
    if rc:
        _lib.check(rc, "tattn_cross_fwd")
    return o, m


def _backward(q, k, v, o, m, lens, do, plan, scale) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    floats, sizes, layouts_of = plan[3:]
    given = q, k, v, o, do
    # Saved tensors come back as hooks on them return them, which need not be the layouts that the forward saw.
    key = q.stride(), k.stride(), v.stride(), o.stride(), do.stride()
    hit = layouts_of.get(key)
    copies = hit[0] if hit else tuple([_tiles_apart(t) for t in given])
    tensors = tuple([aligned(t, c) for t, c in zip(given, copies)])
    q, k, v, o, do = tensors
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    if sizes is None:
        return dq.zero_(), dk.zero_(), dv.zero_()
    m = m.contiguous()
    lens = None if lens is None else lens.contiguous()
    work = m.new_empty(floats)
    in_place = q is given[0] and k is given[1] and v is given[2] and o is given[3] and do is given[4]
    if hit and hit[1] and in_place:
        held = hit[1]
    else:
        held = strides(*tensors, dq, dk, dv)
        if hit is None or in_place:
            remember(layouts_of, key, (copies, held if in_place else None))
    _, st = held
    with _on_device(q):
        rc = _lib.load().tattn_cross_bwd(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), do.data_ptr(), dq.data_ptr(), dk.data_ptr(),
            dv.data_ptr(), m.data_ptr(), None if lens is None else lens.data_ptr(), work.data_ptr(), *st, *sizes, scale,
            _stream(q))
    if rc:
        _lib.check(rc, "tattn_cross_bwd")
    return dq, dk, dv


class _Cross(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, q, k, v, lens, plan, scale):
        o, m = _forward(q, k, v, lens, plan, scale, True)
        ctx.save_for_backward(q, k, v, o, m, lens)
        ctx.args = plan, scale
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, do):
        q, k, v, o, m, lens = ctx.saved_tensors
        return (*_backward(q, k, v, o, m, lens, do, *ctx.args), None, None, None)


def cross_attention(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lens: torch.Tensor | None = None, sm_scale: float | None = None,
) -> torch.Tensor:
    """Attention of every query to all keys of its sequence, of another length: a decoder over an encoder's states, image
    tokens over a text.

    q [batch, heads, queries, dim]; k, v [batch, kv heads, keys, dim]; float16, bfloat16 or float32; heads a multiple of kv
    heads, consecutive heads sharing one; any strides. lens: int32 [batch] on the GPU, keys that the queries of each sequence
    see (clamped to [0, keys]); None: all. What lies at or past them reaches no result and gets zero gradients; a sequence
    without keys gives zeros. sm_scale defaults to 1 / sqrt(dim). Differentiable in q, k and v, with lens too (which must then
    hold the same values when the backward runs); forward-mode derivatives are refused. Gradients of k and v are summed over
    the heads that share them in a fixed order."""
    no_tangents(q, k, v)
    key = layouts(q, k, v, lens)
    plan = _plans.get(key)
    if plan is None:
        plan = remember(_plans, key, _plan(q, k, v, lens))
    scale = float(sm_scale) if sm_scale is not None else 1.0 / math.sqrt(q.shape[3])
    if lens is not None:
        lens = lens.contiguous()
    if (q.requires_grad or k.requires_grad or v.requires_grad) and torch.is_grad_enabled():
        return _Cross.apply(q, k, v, lens, plan, scale)
    return _forward(q, k, v, lens, plan, scale, False)[0]


def _check_prefix(q, prefix_k, prefix_v, k, v, lens, prefix_lens) -> None:
    _check_heads(q, k, v, "k, v")
    _check_heads(q, prefix_k, prefix_v, "prefix_k, prefix_v")
    if k.shape[0] != q.shape[0] or k.shape[1] != prefix_k.shape[1]:
        raise ValueError(f"k, v must have q's batch and the prefix's kv heads, got {k.shape} for {q.shape} and {prefix_k.shape}")
    groups = prefix_k.shape[0]
    if groups < 1 or q.shape[0] % groups:
        raise ValueError(f"the batch must be a multiple of the prefixes, got {q.shape[0]} and {groups}")
    if any(t.dtype != q.dtype for t in (prefix_k, prefix_v, k, v)) or q.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError("q, prefix_k, prefix_v, k, v must share dtype float16 or bfloat16, got "
                         + ", ".join(str(t.dtype) for t in (q, prefix_k, prefix_v, k, v)))
    same_device(q, prefix_k=prefix_k, prefix_v=prefix_v, k=k, v=v, lens=lens, prefix_lens=prefix_lens)
    check_index("lens", lens, torch.int32, (q.shape[0],))
    if prefix_lens is not None:
        check_index("prefix_lens", prefix_lens, torch.int32, (groups,))


_prefix_plans: dict[tuple, tuple] = {}


def _prefix_plan(q, prefix_k, prefix_v, k, v, lens, prefix_lens) -> tuple:
    """Checks a call; which of its tensors are copied, their strides and the output's (None where one is copied), the float32
    values of workspace, and the sizes among the launch's arguments (None: nothing to do)."""
    _check_prefix(q, prefix_k, prefix_v, k, v, lens, prefix_lens)
    _require_gpu(q)
    copies = rows_apart(q), *(t.numel() > 0 and _tiles_apart(t) for t in (prefix_k, prefix_v, k, v))
    if q.numel() == 0:
        return copies, None, 0, None
    z, h, n, d = q.shape
    groups, hk, p = prefix_k.shape[:3]
    sizes = (groups, z // groups, h, hk, n, p, k.shape[2], d)
    out = ctypes.c_int64()
    _lib.check(_lib.load().tattn_prefix_workspace(*sizes, ctypes.byref(out)), "tattn_prefix_workspace")
    held = None if any(copies) else strides(q, prefix_k, prefix_v, k, v, torch.empty_like(q))
    return copies, held, out.value, (*sizes, _DTYPES[q.dtype])


def prefix_attention(
    q: torch.Tensor, prefix_k: torch.Tensor, prefix_v: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lens: torch.Tensor,
    prefix_lens: torch.Tensor | None = None, sm_scale: float | None = None,
) -> torch.Tensor:
    """Attention of the newest tokens of sequences that share a prefix (a system prompt, an image, a prompt that is sampled
    from many times): the prefix is read once for all sequences behind it.

    q [batch, heads, queries, dim]; prefix_k, prefix_v [prefixes, kv heads, prefix, dim]; k, v [batch, kv heads, keys, dim],
    the keys that each sequence added to its prefix; float16 or bfloat16; heads a multiple of kv heads; any strides. The batch
    is a multiple of the prefixes, consecutive sequences sharing one. lens: int32 [batch] on the GPU, keys of its own that
    each sequence holds, the newest included (clamped to [0, keys]); prefix_lens: int32 [prefixes], keys of each prefix (None: all).
    Query n is at position lens - queries + n of its sequence's own keys and sees the whole prefix and its own keys up to its
    position; rows at positions below 0 give zeros. What lies behind the lengths reaches nothing. sm_scale defaults to
    1 / sqrt(dim). For serving: refuses inputs that require gradients or carry forward-mode ones."""
    no_tangents(q, prefix_k, prefix_v, k, v)
    if torch.is_grad_enabled() and (q.requires_grad or prefix_k.requires_grad or prefix_v.requires_grad or k.requires_grad
                                    or v.requires_grad):
        raise ValueError("prefix_attention has no gradients: call it under torch.no_grad()")
    key = layouts(q, prefix_k, prefix_v, k, v, lens, prefix_lens)
    plan = _prefix_plans.get(key)
    if plan is None:
        plan = remember(_prefix_plans, key, _prefix_plan(q, prefix_k, prefix_v, k, v, lens, prefix_lens))
    copies, held, floats, sizes = plan
    pointers = [q.data_ptr(), prefix_k.data_ptr(), prefix_v.data_ptr(), k.data_ptr(), v.data_ptr()]
    if held is None or (pointers[0] | pointers[1] | pointers[2] | pointers[3] | pointers[4]) & 15:
        tensors = [aligned(t, c) for t, c in zip((q, prefix_k, prefix_v, k, v), copies)]
        q, pointers = tensors[0], [t.data_ptr() for t in tensors]
        held = strides(*tensors, torch.empty_like(q))
    o = torch.empty_like(q)
    if sizes is None:
        return o
    lens = lens.contiguous()
    if prefix_lens is not None:
        prefix_lens = prefix_lens.contiguous()
    work = q.new_empty(floats, dtype=torch.float32)
    with _on_device(q):
        rc = _lib.load().tattn_prefix_attention(
            *pointers, o.data_ptr(), None if prefix_lens is None else prefix_lens.data_ptr(), lens.data_ptr(), work.data_ptr(),
            *held[1], *sizes, float(sm_scale) if sm_scale is not None else 1.0 / math.sqrt(q.shape[3]), _stream(q))
    if rc:
        _lib.check(rc, "tattn_prefix_attention")
    return o
