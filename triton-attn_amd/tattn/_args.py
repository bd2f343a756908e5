"""Argument checks and layouts shared by the operators around attention."""

from __future__ import annotations

import torch

from tattn import _lib


def same_device(first: torch.Tensor, **others: torch.Tensor | None) -> None:
    for name, t in others.items():
        if t is not None and t.device != first.device:
            raise ValueError(f"{name} must be on {first.device}, got {t.device}")


def dtype_name(dtype: torch.dtype) -> str:
    return str(dtype).removeprefix("torch.")


def check_index(name: str, t: torch.Tensor, dtype: torch.dtype, shape: tuple) -> None:
    if t.dtype != dtype or tuple(t.shape) != shape:
        raise ValueError(f"{name} must be {dtype_name(dtype)} of shape {list(shape)}, got {dtype_name(t.dtype)} {list(t.shape)}")


def rows(t: torch.Tensor) -> torch.Tensor:
    """t itself where the kernels read its rows (unit d stride, 16-byte aligned), else an aligned contiguous copy."""
    vec = 16 // t.element_size()
    st = t.stride()
    if (st[-1] == 1 or t.shape[-1] <= 1) and t.data_ptr() % 16 == 0:
        for size, s in zip(t.shape[:-1], st):
            if size > 1 and s % vec:
                break
        else:
            return t
    return t.clone(memory_format=torch.contiguous_format)


def strides(*ts: torch.Tensor) -> tuple:
    """An array with each tensor's four strides (missing dimensions and those of one entry have stride 0), to be held
    until the call is made, and the address of each tensor's four."""
    key = tuple(tuple(s if n > 1 else 0 for n, s in zip(t.shape, t.stride())) for t in ts)
    return _lib.stride_rows(key)
