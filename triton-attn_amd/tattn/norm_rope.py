"""Norms of queries and keys for each head, with the position rotation in the same pass.

    q, k = qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions)
    o = attention(q, k, v, causal=True)                              # as many key heads as query heads
    o = window_attention(q, k, v, window=k.shape[2])                 # fewer key heads; or a true window

No counterpart in the reference.
"""

from __future__ import annotations

from typing import Any

import torch
from torch.autograd.function import once_differentiable

from tattn import _lib
from tattn._args import aligned, check_index, layouts, no_tangents, remember, rows, rows_apart, same_device, strides
from tattn.api import _DTYPES, _on_device, _require_gpu, _stream


def _check(q, k, q_weight, k_weight, cos, sin, positions) -> None:
    if q.dim() != 4 or k.dim() != 4 or (q.shape[0], *q.shape[2:]) != (k.shape[0], *k.shape[2:]):
        raise ValueError(f"expected q [batch, heads, seq, dim] and k [batch, kv heads, seq, dim]; got {q.shape}, {k.shape}")
    z, h, n, d = q.shape
    if d not in (16, 32, 64, 128):
        raise ValueError(f"head dim must be 16, 32, 64 or 128, got {d}")
    if h < 1 or k.shape[1] < 1:
        raise ValueError(f"expected at least one head; got {q.shape}, {k.shape}")
    if q.dtype != k.dtype or q.dtype not in _DTYPES:
        raise ValueError(f"q, k must share dtype float16, bfloat16 or float32, got {q.dtype}, {k.dtype}")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if tuple(w.shape) != (d,) or w.dtype != q_weight.dtype or w.dtype not in (q.dtype, torch.float32):
            raise ValueError(f"{name} must have shape [{d}] and be {q.dtype} or float32 (both weights alike), "
                             f"got {list(w.shape)} {w.dtype}")
    if cos.dim() != 2:
        raise ValueError(f"cos must be float32 [positions, {d // 2}], got {list(cos.shape)}")
    check_index("cos", cos, torch.float32, (cos.shape[0], d // 2))
    check_index("sin", sin, torch.float32, tuple(cos.shape))
    if positions is not None:
        check_index("positions", positions, torch.int32, (n,) if positions.dim() == 1 else (z, n))
    elif cos.shape[0] < n:
        raise ValueError(f"cos and sin have {cos.shape[0]} rows for {n} positions")
    if z * n and not cos.shape[0]:
        raise ValueError("cos and sin have no rows")
    same_device(q, k=k, q_weight=q_weight, k_weight=k_weight, cos=cos, sin=sin, positions=positions)


_plans: dict[tuple, tuple] = {}


def _plan(q, k, qw, kw, cos, sin, positions, interleaved) -> tuple:
    """Checks a call; what later calls with these layouts need: which tensors to copy, the strides of inputs and outputs (None
    where q or k is copied), and the sizes among the launch's arguments."""
    _check(q, k, qw, kw, cos, sin, positions)
    _require_gpu(q)
    copies = (rows_apart(q), rows_apart(k), *(not t.is_contiguous() for t in (qw, kw, cos, sin)))
    st = None if copies[0] or copies[1] else strides(q, k, torch.empty_like(q), torch.empty_like(k))
    return copies, st, _scalars(q, k, qw, cos, positions, interleaved)


def _scalars(q, k, qw, cos, positions, interleaved) -> tuple:
    z, h, n, d = q.shape
    pos_stride = n if positions is not None and positions.dim() == 2 else 0
    return pos_stride, z, h, k.shape[1], n, d, cos.shape[0], _DTYPES[q.dtype], _DTYPES[qw.dtype], int(interleaved)


def _forward(q, k, qw, kw, cos, sin, positions, eps, plan) -> tuple[torch.Tensor, torch.Tensor]:
    copies, held, scalars = plan
    q0, k0 = q, k
    q, k = aligned(q, copies[0]), aligned(k, copies[1])
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    if q.numel() == 0:
        return qo, ko
    _, st = held if q is q0 and k is k0 and held else strides(q, k, qo, ko)
    with _on_device(q):
        rc = _lib.load().tattn_norm_rope_fwd(
            q.data_ptr(), k.data_ptr(), qw.data_ptr(), kw.data_ptr(), cos.data_ptr(), sin.data_ptr(),
            None if positions is None else positions.data_ptr(), qo.data_ptr(), ko.data_ptr(), *st, *scalars, eps, _stream(q))
    if rc:
        _lib.check(rc, "tattn_norm_rope_fwd")
    return qo, ko


class _NormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, q, k, qw, kw, cos, sin, positions, eps, plan):
        ctx.save_for_backward(q, k, qw, kw, cos, sin, positions)
        ctx.eps, ctx.scalars = eps, plan[2]
        return _forward(q, k, qw, kw, cos, sin, positions, eps, plan)

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, gq, gk):
        q, k, qw, kw, cos, sin, positions = ctx.saved_tensors
        q, k, gq, gk = rows(q), rows(k), rows(gq), rows(gk)
        dq, dk = torch.empty_like(q), torch.empty_like(k)
        weights = ctx.needs_input_grad[2] or ctx.needs_input_grad[3]
        if q.numel() == 0:
            return dq, dk, torch.zeros_like(qw), torch.zeros_like(kw), None, None, None, None, None
        dqw, dkw, partial = None, None, None
        if weights:
            dqw, dkw = torch.empty_like(qw), torch.empty_like(kw)
            partial = q.new_empty((_lib.NORM_ROPE_ROWS, q.shape[-1]), dtype=torch.float32)
        _, st = strides(q, k, gq, gk, dq, dk)
        with _on_device(q):
            rc = _lib.load().tattn_norm_rope_bwd(
                q.data_ptr(), k.data_ptr(), qw.data_ptr(), kw.data_ptr(), cos.data_ptr(), sin.data_ptr(),
                None if positions is None else positions.data_ptr(), gq.data_ptr(), gk.data_ptr(), dq.data_ptr(),
                dk.data_ptr(), *(None if t is None else t.data_ptr() for t in (dqw, dkw, partial)), *st,
                *ctx.scalars, ctx.eps, _stream(q))
        _lib.check(rc, "tattn_norm_rope_bwd")
        return dq, dk, dqw, dkw, None, None, None, None, None


def qk_norm_rope(
    q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, cos: torch.Tensor,
    sin: torch.Tensor, positions: torch.Tensor | None = None, eps: float = 1e-6, interleaved: bool = False,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Root-mean-square norm of every head of q [batch, heads, seq, dim] and k [batch, kv heads, seq, dim] with the
    weights [dim] (the tensors' dtype, or float32), then the position rotation: pairs (i, i + dim / 2), or (2i, 2i + 1)
    when `interleaved`, turned by the angle with cosine cos[position, i] and sine sin[position, i] (float32
    [any, dim / 2]). positions: int32 [seq] or [batch, seq]; None: 0, 1, ... A position outside the tables gives a row of
    NaN. Outputs keep the order of their input's strides. Differentiable in q, k and both weights (cos and sin get no
    gradients; forward-mode derivatives are refused); float16, bfloat16 or float32, all arithmetic in float32, each result
    rounded once. Any batch, head and sequence strides are read in place."""
    no_tangents(q, k, q_weight, k_weight, cos, sin)
    interleaved = bool(interleaved)
    key = (layouts(q, k, q_weight, k_weight, cos, sin, positions), interleaved)
    plan = _plans.get(key)
    if plan is None:
        plan = remember(_plans, key, _plan(q, k, q_weight, k_weight, cos, sin, positions, interleaved))
    copies = plan[0]
    qw, kw = aligned(q_weight, copies[2]), aligned(k_weight, copies[3])
    cos, sin = aligned(cos, copies[4]), aligned(sin, copies[5])
    if positions is not None:
        positions = positions.contiguous()
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or q_weight.requires_grad or k_weight.requires_grad):
        return _NormRope.apply(q, k, qw, kw, cos, sin, positions, float(eps), plan)
    return _forward(q, k, qw, kw, cos, sin, positions, float(eps), plan)
