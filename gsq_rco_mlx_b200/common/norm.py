"""RMS norms before and after a block, fused with the block's gate, residual scale and sum, and
their vector-Jacobian product.

Between two blocks of a decoder, one call (h the residual stream, y the block's output):

  n  = y / sqrt(mean y^2 + eps) * (w_post + offset)      the norm after the block (optional)
  h' = h + scale * gate * n                                gate: none, per channel, per sequence, per row
  x  = h' / sqrt(mean h'^2 + eps) * (w_pre + offset)      the norm before the next block (optional)

in float32 from the unrounded h', each output rounded once. The general, fused form of the block
engine's gsq_rmsnorm / gsq_rmsnorm_bwd and the residual sums (src/gsq_rco/gsq/e2e.py:90-93,160-174).
"""
from __future__ import annotations

import ctypes as C

import torch

from .. import _lib
from .fp8 import Fp8Tensor, pad16
from .operands import DTYPES, apart, error_word, matrix, on_device, output, row_by_row, \
    same_device, stream_of

MAX_WIDTH = 32768


def _ptr(t):
    return None if t is None else t.data_ptr()


def _weight(w, H, dtype, dev, what):
    if w is None:
        return None
    if w.dtype != dtype or w.shape != (H,):
        raise ValueError(f"{what} must be {dtype} [{H}], got {w.dtype} {tuple(w.shape)}")
    same_device(w, what, dev)
    return w if w.is_contiguous() else w.contiguous()


def _inputs(h, y, w_post, w_pre, gate):
    """(device, h, its pitch, y, its pitch, w_post, w_pre, gate, gate rows), checked."""
    h, ld_h = matrix(h, "h")
    dev, dt = on_device(h, "h"), h.dtype
    T, H = h.shape
    if not H or H > MAX_WIDTH:
        raise ValueError(f"rows of 1 to {MAX_WIDTH} columns, got {H}")
    y, ld_y = matrix(y, "y", T, H, dt)
    same_device(y, "y", dev)
    w_post, w_pre = _weight(w_post, H, dt, dev, "w_post"), _weight(w_pre, H, dt, dev, "w_pre")
    rows = 0
    if gate is not None:
        if gate.dtype != dt or gate.dim() not in (1, 2) or gate.shape[-1] != H:
            raise ValueError(f"gate must be {dt} [{H}] or [rows, {H}], got {gate.dtype} "
                             f"{tuple(gate.shape)}")
        same_device(gate, "gate", dev)
        gate = gate if gate.is_contiguous() else gate.contiguous()
        rows = 1 if gate.dim() == 1 else gate.shape[0]
        if not rows or T % rows:
            raise ValueError(f"{rows} gate rows do not divide {T} rows")
    return dev, h, ld_h, y, ld_y, w_post, w_pre, gate, rows


def residual_norm(h, y, w_post=None, w_pre=None, gate=None, scale=1.0, eps=1e-6, offset=0.0,
                  fp8=False, out=None):
    """(h', x, stats) of rows h, y [T, H] (bf16, float16 or float32; rows may be strided), weights
    [H] and gate [H] or [rows, H] of the same type; gate row i serves the rows [i T / rows,
    (i + 1) T / rows). x is None without w_pre; with fp8 an Fp8Tensor (x in e4m3 with a scale per
    row and 128 columns: what Fp8Linear takes). stats float32 [2, T]: the reciprocal root mean
    squares of y and h' (1 where there is no norm), for residual_norm_vjp. out: where h' goes (h
    itself for a residual stream updated in place; no other overlap with h, y or the parameters)."""
    dev, h, ld_h, y, ld_y, w_post, w_pre, gate, rows = _inputs(h, y, w_post, w_pre, gate)
    if fp8 and w_pre is None:
        raise ValueError("fp8 needs w_pre (x is what is quantized)")
    T, H = h.shape
    dt = h.dtype
    h2, ld_h2 = output(out, T, H, dt, h, "out")
    if out is not None:
        row_by_row(out, ld_h2, h, ld_h, "out", "h")
        row_by_row(out, ld_h2, y, ld_y, "out", "y")
        for w, name in ((w_post, "w_post"), (w_pre, "w_pre"), (gate, "gate")):
            if w is not None:
                apart(out, "out", w, name)
    stats = h.new_empty((2, T), dtype=torch.float32)
    x, xp, codes, scales, ld_c = None, None, None, None, 0
    if fp8:
        x = Fp8Tensor.empty(T, H, h.device)
        codes, scales, ld_c = x.codes.data_ptr(), x.scales.data_ptr(), pad16(H)
    elif w_pre is not None:
        x = h.new_empty((T, H))
        xp = x.data_ptr()
    if T:
        _lib.call("gsq_residual_norm", h.data_ptr(), ld_h, y.data_ptr(), ld_y, _ptr(w_post),
                  _ptr(w_pre), _ptr(gate), rows, T, H, DTYPES[dt], float(scale),
                  float(eps), float(offset), h2.data_ptr(), ld_h2, xp, H, codes, ld_c, scales, T, stats.data_ptr(),
                  stream_of(dev))
    return h2, x, stats


def residual_norm_vjp(h, y, w_post, w_pre, stats, dh, dx, gate=None, scale=1.0, offset=0.0):
    """Gradients of residual_norm at its inputs for the cotangents dh of h' (None: zero) and dx of
    x (None without w_pre): a dict of dh, dy (in the rows' type) and the float32 dw_post [H],
    dw_pre [H], dgate (the gate's shape), None for the absent ones. stats: of the forward pass.
    The sums over rows run in a fixed order: the same inputs give the same bits."""
    dev, h, ld_h, y, ld_y, w_post, w_pre, gate, rows = _inputs(h, y, w_post, w_pre, gate)
    T, H = h.shape
    dt = h.dtype
    if stats.dtype != torch.float32 or stats.shape != (2, T):
        raise ValueError(f"stats must be float32 [2, {T}], got {stats.dtype} {tuple(stats.shape)}")
    same_device(stats, "stats", dev)
    stats = stats.contiguous()
    if (dx is None) != (w_pre is None):
        raise ValueError("dx comes with w_pre, and only with it")
    if dh is None and dx is None:
        raise ValueError("dh or dx is needed")
    ld_dh = ld_dx = 0
    if dh is not None:
        dh, ld_dh = matrix(dh, "dh", T, H, dt)
        same_device(dh, "dh", dev)
    if dx is not None:
        dx, ld_dx = matrix(dx, "dx", T, H, dt)
        same_device(dx, "dx", dev)
    f32 = torch.float32
    make = h.new_empty if T else h.new_zeros
    g = {"dh": h.new_empty((T, H)), "dy": h.new_empty((T, H)),
         "dw_post": None if w_post is None else make((H,), dtype=f32),
         "dw_pre": None if w_pre is None else make((H,), dtype=f32),
         "dgate": None if gate is None else make(gate.shape, dtype=f32)}
    if not T:
        return g
    n = C.c_int64()
    _lib.check(_lib.lib().gsq_residual_norm_bwd_workspace(T, H, DTYPES[dt], rows, C.byref(n)),
               "gsq_residual_norm_bwd_workspace")
    # allocated per call on the calling stream: nothing is shared between calls
    ws = h.new_empty((n.value,), dtype=torch.uint8)
    _lib.call("gsq_residual_norm_bwd", h.data_ptr(), ld_h, y.data_ptr(), ld_y, _ptr(w_post),
              _ptr(w_pre), _ptr(gate), rows, stats.data_ptr(), _ptr(dh), ld_dh, _ptr(dx), ld_dx, T,
              H, DTYPES[dt], float(scale), float(offset), g["dh"].data_ptr(), H, g["dy"].data_ptr(), H,
              _ptr(g["dw_post"]), _ptr(g["dw_pre"]), _ptr(g["dgate"]), ws.data_ptr(), n.value,
              error_word(h.device).data_ptr(), stream_of(dev))
    return g
