"""Checks of tensor arguments shared by the operators that take bf16, float16 and float32. They run
on every call of operators that take a few microseconds on the GPU, so they ask each tensor once
and build messages only to raise them."""
from __future__ import annotations

import numpy as np
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


def runs(t):
    """Where t [..., C] lies whose last dimension is contiguous: (address, [(bytes from one to the
    next, how many), ...] of the other dimensions, widest first, bytes of a run of C)."""
    n = t.element_size()
    dims = [(s * n, c) for s, c in zip(t.stride()[:-1], t.shape[:-1]) if c > 1]
    dims.sort(reverse=True)
    return t.data_ptr(), dims, t.shape[-1] * n


def _extent(dims, width):
    return width + sum((c - 1) * s for s, c in dims)


def _surely_apart(da, wa, db, wb, d):
    """Whether runs of `da`, `wa` at 0 and of `db`, `wb` at d have no byte in common, by their
    extents: as a whole, or inside a step that both repeat."""
    if d >= _extent(da, wa) or -d >= _extent(db, wb):
        return True
    for s, _ in da:
        if s and any(s == x for x, _ in db):
            ia, ib = [x for x in da if x[0] != s], [x for x in db if x[0] != s]
            if _extent(ia, wa) <= s and _extent(ib, wb) <= s:
                # bytes in common are so many whole steps apart as bring b to d mod s or s before
                return _surely_apart(ia, wa, ib, wb, d % s) and \
                    _surely_apart(ia, wa, ib, wb, d % s - s)
    return False


def box(t):
    """Where t [T, n, C] lies, in bytes: (address, the wider step, what lies inside it, the whole
    extent, whether its runs of C are one behind the other as this says). None: nowhere."""
    if t is None:
        return 0, 0, 0, 0, True
    T, n, C = t.shape
    st, sh, _ = t.stride()
    e = t.element_size()
    if T == 1 or n > 1 and sh > st:
        st, T, sh, n = sh, n, st, T
    if T == 1:
        st = 0
    inner = (n - 1) * sh + C if n > 1 else C
    return (t.data_ptr(), st * e, inner * e, ((T - 1) * st + inner) * e,
            (T == 1 or st >= inner) and (n == 1 or sh >= C))


def same_rows(a, b):
    """Whether tensors of one shape and type are the same elements in the same places."""
    if a.data_ptr() != b.data_ptr():
        return False
    s, t = a.stride(), b.stride()
    return s == t or all(x == y for x, y, c in zip(s, t, a.shape) if c > 1)


def boxes_apart(a, b):
    """Whether two boxes have no byte in common as far as these figures show it."""
    d = b[0] - a[0]
    return d >= a[3] or -d >= b[3] or a[1] == b[1] and b[2] <= a[1] and \
        a[2] <= d % a[1] <= a[1] - b[2]


_MOST_RUNS = 1 << 22   # that are compared one by one


def _starts(dims):
    at = np.zeros(1, np.int64)
    for s, c in dims:
        at = (at[:, None] + s * np.arange(c, dtype=np.int64)).reshape(-1)
    return np.sort(at)


def _count(dims):
    n = 1
    for _, c in dims:
        n *= c
    return n


def meet(a, b):
    """Whether two sets of runs have a byte in common (True also for more runs than are compared
    one by one, where the extents do not settle it)."""
    (pa, da, wa), (pb, db, wb) = a, b
    if _surely_apart(da, wa, db, wb, pb - pa):
        return False
    if max(_count(da), _count(db)) > _MOST_RUNS:
        return True
    A, B = _starts(da), _starts(db) + (pb - pa)
    i = np.searchsorted(A, B - wa, "right")   # the first run of a that ends behind b's start
    return bool(np.any(A[np.minimum(i, len(A) - 1)][i < len(A)] < B[i < len(A)] + wb))


def apart(a, what, b, name):
    """Refuses a that has a byte in common with b (rows whose elements are contiguous)."""
    d, n = b.data_ptr() - a.data_ptr(), a.element_size()
    if a.is_contiguous() and d >= a.numel() * n or b.is_contiguous() and \
            -d >= b.numel() * b.element_size() or not a.numel() or not b.numel():
        return
    if meet(runs(a), runs(b)):
        raise ValueError(f"{what} overlaps {name}")


def repeats(a):
    """Whether runs lie over one another (True also where it is not settled, as in meet)."""
    _, dims, width = a
    room = width
    for s, c in reversed(dims):
        if s < room:
            if _count(dims) > _MOST_RUNS:
                return True
            at = _starts(dims)
            return bool(np.any(at[1:] - at[:-1] < width))
        room += (c - 1) * s
    return False
