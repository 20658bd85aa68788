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
from ..gemm import err_flag
from .fp8 import Fp8Tensor, pad16
from .operands import DTYPES, matrix, on_device, output, pitch

MAX_WIDTH = 32768


def _ptr(t):
    return None if t is None else t.data_ptr()


def _weight(w, H, dtype, what):
    if w is None:
        return None
    if w.dtype != dtype or tuple(w.shape) != (H,):
        raise ValueError(f"{what} must be {dtype} [{H}], got {w.dtype} {tuple(w.shape)}")
    on_device(w, what)
    return w.contiguous()


def _inputs(h, y, w_post, w_pre, gate):
    h = matrix(h, "h")
    T, H = h.shape
    if not H or H > MAX_WIDTH:
        raise ValueError(f"rows of 1 to {MAX_WIDTH} columns, got {H}")
    y = matrix(y, "y", T, H, h.dtype)
    w_post, w_pre = _weight(w_post, H, h.dtype, "w_post"), _weight(w_pre, H, h.dtype, "w_pre")
    rows = 0
    if gate is not None:
        if gate.dtype != h.dtype or gate.dim() not in (1, 2) or gate.shape[-1] != H:
            raise ValueError(f"gate must be {h.dtype} [{H}] or [rows, {H}], got {gate.dtype} "
                             f"{tuple(gate.shape)}")
        on_device(gate, "gate")
        gate = gate.contiguous()
        rows = 1 if gate.dim() == 1 else gate.shape[0]
        if not rows or T % rows:
            raise ValueError(f"{rows} gate rows do not divide {T} rows")
    return h, y, w_post, w_pre, gate, rows


def residual_norm(h, y, w_post=None, w_pre=None, gate=None, scale=1.0, eps=1e-6, offset=0.0,
                  fp8=False, out=None):
    """(h', x, stats) of rows h, y [T, H] (bf16, float16 or float32; rows may be strided), weights
    [H] and gate [H] or [rows, H] of the same type; gate row i serves the rows [i T / rows,
    (i + 1) T / rows). x is None without w_pre; with fp8 an Fp8Tensor (x in e4m3 with a scale per
    row and 128 columns: what Fp8Linear takes). stats float32 [2, T]: the reciprocal root mean
    squares of y and h' (1 where there is no norm), for residual_norm_vjp. out: where h' goes (h
    itself for a residual stream updated in place)."""
    h, y, w_post, w_pre, gate, rows = _inputs(h, y, w_post, w_pre, gate)
    if fp8 and w_pre is None:
        raise ValueError("fp8 needs w_pre (x is what is quantized)")
    T, H = h.shape
    dev, dt = h.device, h.dtype
    h2 = output(out, T, H, dt, dev, "out")
    stats = torch.empty(2, T, device=dev, dtype=torch.float32)
    x = None
    if w_pre is not None:
        x = Fp8Tensor.empty(T, H, dev) if fp8 else torch.empty(T, H, device=dev, dtype=dt)
    if T:
        codes = x.codes if fp8 else None
        _lib.call("gsq_residual_norm", h.data_ptr(), pitch(h), y.data_ptr(), pitch(y),
                  _ptr(w_post), _ptr(w_pre), _ptr(gate), rows, T, H, DTYPES[dt], float(scale),
                  float(eps), float(offset), h2.data_ptr(), pitch(h2),
                  None if fp8 else _ptr(x), H, _ptr(codes), pad16(H),
                  x.scales.data_ptr() if fp8 else None, T, stats.data_ptr(), _lib.stream_ptr())
    return h2, x, stats


def residual_norm_vjp(h, y, w_post, w_pre, stats, dh, dx, gate=None, scale=1.0, offset=0.0):
    """Gradients of residual_norm at its inputs for the cotangents dh of h' (None: zero) and dx of
    x (None without w_pre): a dict of dh, dy (in the rows' type) and the float32 dw_post [H],
    dw_pre [H], dgate (the gate's shape), None for the absent ones. stats: of the forward pass.
    The sums over rows run in a fixed order: the same inputs give the same bits."""
    h, y, w_post, w_pre, gate, rows = _inputs(h, y, w_post, w_pre, gate)
    T, H = h.shape
    dev, dt = h.device, h.dtype
    if stats.dtype != torch.float32 or tuple(stats.shape) != (2, T):
        raise ValueError(f"stats must be float32 [2, {T}], got {stats.dtype} {tuple(stats.shape)}")
    on_device(stats, "stats")
    stats = stats.contiguous()
    if (dx is None) != (w_pre is None):
        raise ValueError("dx comes with w_pre, and only with it")
    if dh is None and dx is None:
        raise ValueError("dh or dx is needed")
    dh = None if dh is None else matrix(dh, "dh", T, H, dt)
    dx = None if dx is None else matrix(dx, "dx", T, H, dt)
    f32 = {"device": dev, "dtype": torch.float32}
    make = torch.empty if T else torch.zeros
    g = {"dh": torch.empty(T, H, device=dev, dtype=dt),
         "dy": torch.empty(T, H, device=dev, dtype=dt),
         "dw_post": None if w_post is None else make(H, **f32),
         "dw_pre": None if w_pre is None else make(H, **f32),
         "dgate": None if gate is None else make(gate.shape, **f32)}
    if not T:
        return g
    n = C.c_int64()
    _lib.check(_lib.lib().gsq_residual_norm_bwd_workspace(T, H, DTYPES[dt], rows, C.byref(n)),
               "gsq_residual_norm_bwd_workspace")
    # allocated per call on the calling stream: nothing is shared between calls
    ws = torch.empty(n.value, device=dev, dtype=torch.uint8)
    _lib.call("gsq_residual_norm_bwd", h.data_ptr(), pitch(h), y.data_ptr(), pitch(y),
              _ptr(w_post), _ptr(w_pre), _ptr(gate), rows, stats.data_ptr(), _ptr(dh),
              0 if dh is None else pitch(dh), _ptr(dx), 0 if dx is None else pitch(dx), T, H,
              DTYPES[dt], float(scale), float(offset), g["dh"].data_ptr(), H, g["dy"].data_ptr(),
              H, _ptr(g["dw_post"]), _ptr(g["dw_pre"]), _ptr(g["dgate"]), ws.data_ptr(),
              ws.numel(), err_flag(dev).data_ptr(), _lib.stream_ptr())
    return g
