"""Rotation of queries and keys by positions on several axes, for tokens of images and video among those of text.

    q, k = qk_rope_axes(q, k, cos, sin, positions, axes=(0,) * 16 + (1,) * 24 + (2,) * 24)     # time, height, width
    q, k = qk_rope_axes(..., q_weight=qw, k_weight=kw)                                         # norms of the heads first

No counterpart in the reference.
"""

from __future__ import annotations

import ctypes
from typing import Any, Sequence

import torch
from torch.autograd.function import once_differentiable

from tattn import _lib
from tattn._args import aligned, check_index, layouts, no_tangents, remember, rows, rows_apart, same_device, strides, whole
from tattn.api import _DTYPES, _on_device, _require_gpu, _stream
from tattn.norm_rope import _check as _check_norm_rope


def _check(q, k, q_weight, k_weight, cos, sin, positions, axes) -> None:
    if (q_weight is None) != (k_weight is None):
        raise ValueError("give both q_weight and k_weight, or neither")
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError(f"expected q [batch, heads, seq, dim] and k [batch, kv heads, seq, dim]; got {q.shape}, {k.shape}")
    z, _, n, d = q.shape
    if positions.dim() not in (2, 3) or not 1 <= positions.shape[0] <= 8:
        raise ValueError(f"positions must be int32 [axes, seq] or [axes, batch, seq] with 1 to 8 axes, got {list(positions.shape)}")
    count = positions.shape[0]
    check_index("positions", positions, torch.int32, (count, n) if positions.dim() == 2 else (count, z, n))
    same_device(q, positions=positions)
    # The rest as the norm and the rotation on one axis, for which the stand-ins' position is any row of the tables.
    weight = q.new_empty(d) if q_weight is None else None
    _check_norm_rope(q, k, weight if q_weight is None else q_weight, weight if k_weight is None else k_weight, cos, sin,
                     positions[0])
    if len(axes) != d // 2 or any(not -1 <= a < count for a in axes):
        raise ValueError(f"axes must hold {d // 2} numbers from -1 to {count - 1}, one for each pair, got {list(axes)}")


_plans: dict[tuple, tuple] = {}


def _plan(q, k, qw, kw, cos, sin, positions, axes, interleaved) -> tuple:
    """Checks a call; what later calls with these layouts need: which tensors to copy, the strides of inputs and outputs (None
    where q or k is copied), the axes as the library reads them, and the sizes among the launch's arguments."""
    _check(q, k, qw, kw, cos, sin, positions, axes)
    _require_gpu(q)
    copies = (rows_apart(q), rows_apart(k), *(t is not None and not t.is_contiguous() for t in (qw, kw, cos, sin)))
    st = None if copies[0] or copies[1] else strides(q, k, torch.empty_like(q), torch.empty_like(k))
    z, h, n, d = q.shape
    deep = positions.dim() == 3
    sizes = (positions.shape[0], z * n if deep else n, n if deep else 0, z, h, k.shape[1], n, d, cos.shape[0], _DTYPES[q.dtype],
             _DTYPES[q.dtype if qw is None else qw.dtype], int(interleaved))
    return copies, st, (ctypes.c_int32 * len(axes))(*axes), sizes


def _pointer(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _forward(q, k, qw, kw, cos, sin, positions, eps, plan) -> tuple[torch.Tensor, torch.Tensor]:
    copies, held, axes, sizes = plan
    q0, k0 = q, k
    q, k = aligned(q, copies[0]), aligned(k, copies[1])
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    if q.numel() == 0:
        return qo, ko
    _, st = held if held and q is q0 and k is k0 else strides(q, k, qo, ko)
    with _on_device(q):
        rc = _lib.load().tattn_rope_axes_fwd(
            q.data_ptr(), k.data_ptr(), _pointer(qw), _pointer(kw), cos.data_ptr(), sin.data_ptr(), positions.data_ptr(), axes,
            qo.data_ptr(), ko.data_ptr(), *st, *sizes, eps, _stream(q))
    if rc:
        _lib.check(rc, "tattn_rope_axes_fwd")
    return qo, ko


class _RopeAxes(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, q, k, qw, kw, cos, sin, positions, eps, plan):
        # Without norms the gradients need only the angles.
        ctx.save_for_backward(*((None, None) if qw is None else (q, k)), qw, kw, cos, sin, positions)
        ctx.eps, ctx.axes, ctx.sizes = eps, plan[2], plan[3]
        return _forward(q, k, qw, kw, cos, sin, positions, eps, plan)

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, gq, gk):
        # Saved tensors come back as hooks on them return them, which need not be in the layouts that were saved.
        q, k, *rest = ctx.saved_tensors
        qw, kw, cos, sin, positions = (t if t is None else aligned(t, not t.is_contiguous()) for t in rest)
        gq, gk = rows(gq), rows(gk)
        norm = qw is not None
        q, k = (rows(q), rows(k)) if norm else (gq, gk)
        dq, dk = torch.empty_like(q), torch.empty_like(k)
        weights = norm and (ctx.needs_input_grad[2] or ctx.needs_input_grad[3])
        if q.numel() == 0:
            return dq, dk, *((torch.zeros_like(qw), torch.zeros_like(kw)) if norm else (None, None)), *[None] * 5
        dqw, dkw, partial = None, None, None
        if weights:
            dqw, dkw = torch.empty_like(qw), torch.empty_like(kw)
            partial = q.new_empty((_lib.NORM_ROPE_ROWS, q.shape[-1]), dtype=torch.float32)
        _, st = strides(q, k, gq, gk, dq, dk)
        with _on_device(gq):
            rc = _lib.load().tattn_rope_axes_bwd(
                _pointer(q), _pointer(k), _pointer(qw), _pointer(kw), cos.data_ptr(), sin.data_ptr(), positions.data_ptr(),
                ctx.axes, gq.data_ptr(), gk.data_ptr(), dq.data_ptr(), dk.data_ptr(), _pointer(dqw), _pointer(dkw),
                _pointer(partial), *st, *ctx.sizes, ctx.eps, _stream(gq))
        if rc:
            _lib.check(rc, "tattn_rope_axes_bwd")
        return dq, dk, dqw, dkw, *[None] * 5


def qk_rope_axes(
    q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor, axes: Sequence[int],
    interleaved: bool = False, q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Rotation of every head of q [batch, heads, seq, dim] and k [batch, kv heads, seq, dim] by positions on up to eight axes:
    pair i, elements (i, i + dim / 2), or (2i, 2i + 1) when `interleaved`, is turned by the angle with cosine cos[x, i] and sine
    sin[x, i] (float32 [any, dim / 2]), x being the token's position on axis axes[i]. positions: int32 [axes, seq] or [axes,
    batch, seq]. axes: dim / 2 whole numbers; -1 leaves a pair as it is. A position outside the tables makes the pairs of its
    axis NaN. With both weights [dim] (the tensors' dtype, or float32) the root-mean-square norm of every head comes first, as in
    qk_norm_rope. Outputs keep the order of their input's strides. Differentiable in q, k and the weights (cos and sin get no
    gradients; forward-mode derivatives are refused); float16, bfloat16 or float32, all arithmetic in float32, each result
    rounded once. Any batch, head and sequence strides are read in place."""
    no_tangents(q, k, q_weight, k_weight, cos, sin)
    interleaved = bool(interleaved)
    axes = tuple(axes)
    if set(map(type, axes)) != {int}:
        axes = tuple([whole("axis", a) for a in axes])
    key = (layouts(q, k, q_weight, k_weight, cos, sin, positions), axes, interleaved)
    plan = _plans.get(key)
    if plan is None:
        plan = remember(_plans, key, _plan(q, k, q_weight, k_weight, cos, sin, positions, axes, interleaved))
    copies = plan[0]
    qw, kw = (t if t is None else aligned(t, c) for t, c in ((q_weight, copies[2]), (k_weight, copies[3])))
    cos, sin = aligned(cos, copies[4]), aligned(sin, copies[5])
    positions = positions.contiguous()
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or qw is not None and (qw.requires_grad or kw.requires_grad)):
        return _RopeAxes.apply(q, k, qw, kw, cos, sin, positions, float(eps), plan)
    return _forward(q, k, qw, kw, cos, sin, positions, float(eps), plan)
