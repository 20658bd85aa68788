"""Checks of tensor arguments shared by the operators that take bf16, float16 and float32."""
from __future__ import annotations

import torch

DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def on_device(t, what):
    """t is on the current CUDA device (where the launch and its stream are)."""
    if not t.is_cuda:
        raise ValueError(f"{what} must be a CUDA tensor")
    if t.get_device() != torch.cuda.current_device():
        raise ValueError(f"{what} is on {t.device}, the current device is "
                         f"cuda:{torch.cuda.current_device()}")


def matrix(t, what, rows=None, cols=None, dtype=None):
    """t as a matrix whose rows are contiguous (strided rows are taken as they are, any other
    layout is copied)."""
    if t.dim() != 2 or t.dtype not in DTYPES:
        raise ValueError(f"{what} must be a bf16, float16 or float32 matrix, got {t.dtype} "
                         f"{tuple(t.shape)}")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{what} must be {dtype}, got {t.dtype}")
    if (rows is not None and t.shape[0] != rows) or (cols is not None and t.shape[1] != cols):
        raise ValueError(f"{what} must be [{'any' if rows is None else rows}, "
                         f"{'any' if cols is None else cols}], got {tuple(t.shape)}")
    on_device(t, what)
    if t.stride(1) != 1 and t.shape[1] > 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        t = t.contiguous()
    return t


def pitch(t):
    """Elements between the rows of a matrix (one row: any number that holds it)."""
    return max(t.stride(0), t.shape[1])


def output(out, rows, cols, dtype, dev, what):
    """out, checked, or a new matrix."""
    if out is None:
        return torch.empty(rows, cols, device=dev, dtype=dtype)
    if out.dtype != dtype or tuple(out.shape) != (rows, cols):
        raise ValueError(f"{what} must be {dtype} [{rows}, {cols}]")
    on_device(out, what)
    if cols > 1 and out.stride(1) != 1 or rows > 1 and out.stride(0) < cols:
        raise ValueError(f"{what} must have contiguous rows that do not overlap")
    return out
