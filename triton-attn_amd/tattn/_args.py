"""Argument checks and layouts shared by the operators around attention."""

from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad


def same_device(first: torch.Tensor, **others: torch.Tensor | None) -> None:
    for name, t in others.items():
        if t is not None and t.device != first.device:
            raise ValueError(f"{name} must be on {first.device}, got {t.device}")


def dtype_name(dtype: torch.dtype) -> str:
    return str(dtype).removeprefix("torch.")


def no_tangents(*ts: torch.Tensor | None) -> None:
    """Refuses dual tensors: the kernels would lose their tangents. Outside a level of forward-mode AD there are none."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in ts):
        raise ValueError("no forward-mode derivatives: the tensors must not carry tangents")


def whole(name: str, x) -> int:
    """x's value now as a plain int, fit to be kept in a key: numbers of other types, and tensors, may change or compare by identity."""
    if type(x) is int:
        return x
    try:
        n = int(x)
    except (TypeError, ValueError):
        n = None
    if n is None or n != x:
        raise ValueError(f"{name} must be a whole number, got {x!r}")
    return n


def check_index(name: str, t: torch.Tensor, dtype: torch.dtype, shape: tuple) -> None:
    if t.dtype != dtype or tuple(t.shape) != shape:
        raise ValueError(f"{name} must be {dtype_name(dtype)} of shape {list(shape)}, got {dtype_name(t.dtype)} {list(t.shape)}")


def rows_apart(t: torch.Tensor) -> bool:
    """Whether the kernels cannot read t's rows where they lie: unit d stride, strides of whole 16-byte chunks."""
    vec, st = 16 // t.element_size(), t.stride()
    return st[-1] != 1 or any(size > 1 and s % vec for size, s in zip(t.shape[:-1], st))


def rows(t: torch.Tensor) -> torch.Tensor:
    """t itself where the kernels read its rows, else an aligned contiguous copy."""
    return aligned(t, rows_apart(t))


def layouts(*ts: torch.Tensor | None) -> tuple:
    """What the checks of a call and its launch arguments depend on, but for the data's addresses."""
    return tuple([None if t is None else (t.shape, t.stride(), t.dtype, t.device) for t in ts])


def remember(plans: dict, key: tuple, plan: tuple) -> tuple:
    """Keeps what the checks of a call made of its tensors' layouts, for calls with the same ones."""
    if len(plans) >= 1024:
        plans.clear()
    plans[key] = plan
    return plan


def aligned(t: torch.Tensor, copy: bool) -> torch.Tensor:
    """t, or an aligned contiguous copy where its layout asks for one or its data does not start on 16 bytes."""
    return t.clone(memory_format=torch.contiguous_format) if copy or t.data_ptr() & 15 else t


_stride_arrays: dict[tuple, tuple] = {}


def strides(*ts: torch.Tensor) -> tuple:
    """An array with each tensor's four strides (missing dimensions and those of one entry have stride 0), to be held
    until the call is made, and the address of each tensor's four."""
    key = tuple([(t.shape, t.stride()) for t in ts])
    hit = _stride_arrays.get(key)
    if hit is None:
        flat = [s for shape, st in key for s in ([s if n > 1 else 0 for n, s in zip(shape, st)] + [0] * 4)[:4]]
        arr = (ctypes.c_int64 * len(flat))(*flat)
        base = ctypes.addressof(arr)
        hit = remember(_stride_arrays, key, (arr, [base + 32 * i for i in range(len(ts))]))
    return hit
