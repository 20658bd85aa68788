"""Checks of tensor arguments shared by the operators that take bf16, float16 and float32. They run
on every call of operators that take a few microseconds on the GPU, so they ask each tensor once
and build messages only to raise them."""
from __future__ import annotations

import torch

from .. import gemm

MAX_DIM = 1 << 30   # rows or columns of an operand (32-bit counts in the kernels)
DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def on_device(t, what):
    """The index of the current CUDA device, where t has to be (there are the launch and its
    stream)."""
    d = t.get_device()
    if d < 0:
        raise ValueError(f"{what} must be a CUDA tensor")
    if d != torch._C._cuda_getDevice():
        raise ValueError(f"{what} is on {t.device}, the current device is "
                         f"cuda:{torch.cuda.current_device()}")
    return d


def same_device(t, what, dev):
    """t is on device `dev` (of on_device)."""
    if t.get_device() != dev:
        raise ValueError(f"{what} must be on cuda:{dev}, got {t.device}")


def stream_of(dev):
    """The current stream's handle on device `dev`."""
    return torch._C._cuda_getCurrentRawStream(dev)


def error_word(device):
    """The device's error word of bounded waits (gemm.check_err). Made during a capture it would be
    cleared by every replay, and with it an error that another call left."""
    if device not in gemm._ERR and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("the first call on a device cannot be captured: make one before")
    return gemm.err_flag(device)


def matrix(t, what, rows=None, cols=None, dtype=None):
    """t as a matrix whose rows are contiguous (strided rows are taken as they are, any other
    layout is copied), and the elements between its rows. The caller checks its device."""
    if t.dim() != 2 or t.dtype not in DTYPES:
        raise ValueError(f"{what} must be a bf16, float16 or float32 matrix, got {t.dtype} "
                         f"{tuple(t.shape)}")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{what} must be {dtype}, got {t.dtype}")
    r, c = t.shape
    if rows is not None and r != rows or cols is not None and c != cols:
        raise ValueError(f"{what} must be [{'any' if rows is None else rows}, "
                         f"{'any' if cols is None else cols}], got {tuple(t.shape)}")
    if r > MAX_DIM or c > MAX_DIM:
        raise ValueError(f"{what} has more than {MAX_DIM} rows or columns: {tuple(t.shape)}")
    s0, s1 = t.stride()
    if s1 != 1 and c > 1 or s0 < c and r > 1:
        t = t.contiguous()
        s0 = c
    return t, s0 if s0 > c else c


def output(out, rows, cols, dtype, like, what):
    """out, checked, or a new matrix beside `like`; and the elements between its rows."""
    if out is None:
        return like.new_empty((rows, cols), dtype=dtype), cols
    if out.dtype != dtype or tuple(out.shape) != (rows, cols):
        raise ValueError(f"{what} must be {dtype} [{rows}, {cols}]")
    same_device(out, what, like.get_device())
    s0, s1 = out.stride()
    if s1 != 1 and cols > 1 or s0 < cols and rows > 1:
        raise ValueError(f"{what} must have contiguous rows that do not overlap")
    return out, s0 if s0 > cols else cols


def row_by_row(out, ld_out, x, ld_x, what, name):
    """out [rows, cols] is x's own rows, or shares no element with x (of the same type and shape):
    what a kernel that reads and writes row by row may be given."""
    rows, cols = x.shape
    d = out.data_ptr() - x.data_ptr()
    if not rows or d == 0 and (ld_out == ld_x or rows == 1):
        return
    n = x.element_size()
    if d >= ((rows - 1) * ld_x + cols) * n or -d >= ((rows - 1) * ld_out + cols) * n:
        return
    # columns of one wider buffer
    if ld_out == ld_x and cols * n <= d % (ld_x * n) <= (ld_x - cols) * n:
        return
    raise ValueError(f"{what} overlaps {name} without being the same rows")
