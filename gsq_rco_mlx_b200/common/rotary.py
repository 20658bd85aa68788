"""Rotary positions of q and k: half and interleaved layouts, part of the head, frequencies
scaled for contexts longer than the model was trained on, any positions; and their
vector-Jacobian product.

The general form of the block engine's rotation (gsq/e2e.py rope_tables / gsq_rope_split: half
layout, heads of 64, positions 0..T-1, src/gsq_rco/gsq/e2e.py:96-108). Pair j of a head at
position p turns by the angle p w_j, w_j = theta^(-2 j / rotary_dim) before scaling:

  half          pairs (j, j + rotary_dim / 2)        interleaved   pairs (2 j, 2 j + 1)

scaling (a dict with "type" and "factor" f >= 1):
  "linear"  w_j / f (position interpolation)
  "ntk"     theta -> theta f^(d / (d - 2)), d = rotary_dim: the fastest pair unchanged, the slowest
            one stretched by f
  "yarn"    with "original" (the trained context L): w_j / f for the slow pairs, w_j for the fast
            ones, a ramp over j between the pairs that turn "slow" (1) and "fast" (32) times in L;
            cos and sin times "attention" (default 0.1 ln f + 1)
  "bands"   with "original" L, "low" (1) and "high" (4): w_j / f below `low` turns in L, w_j above
            `high`, linear in the number of turns between
"""
from __future__ import annotations

import math

import numpy as np
import torch

from .. import _lib
from .operands import DTYPES, box, boxes_apart, meet, on_device, repeats, runs, same_device, \
    same_rows, stream_of

MAX_HEADS = 65536
_KEYS = {"linear": set(), "ntk": set(), "yarn": {"original", "slow", "fast", "attention"},
         "bands": {"original", "low", "high"}}


def frequencies(rotary_dim, theta=1e6, scaling=None):
    """(w float64 [rotary_dim / 2], the factor on cos and sin)."""
    d = int(rotary_dim)
    j = np.arange(0, d, 2, dtype=np.float64)
    w = float(theta) ** (-j / d)
    if scaling is None:
        return w, 1.0
    kind = scaling.get("type")
    if kind not in _KEYS:
        raise ValueError(f"unknown scaling type {kind!r}: one of {', '.join(_KEYS)}")
    extra = set(scaling) - {"type", "factor"} - _KEYS[kind]
    if extra:
        raise ValueError(f"scaling {kind!r} does not take {sorted(extra)}")
    f = float(scaling.get("factor", 0.0))
    if not (f >= 1.0 and math.isfinite(f)):
        raise ValueError(f"scaling factor must be a finite number >= 1, got {f}")
    if kind == "linear":
        return w / f, 1.0
    if kind == "ntk":
        return (float(theta) * f ** (d / max(1, d - 2))) ** (-j / d), 1.0
    L = float(scaling.get("original", 0))
    if not (L > 0 and math.isfinite(L)):
        raise ValueError(f"scaling {kind!r} needs 'original', the trained context length")
    if kind == "yarn":
        slow, fast = float(scaling.get("slow", 1.0)), float(scaling.get("fast", 32.0))
        if not 0 < slow < fast:
            raise ValueError(f"expected 0 < slow < fast, got {slow}, {fast}")
        # the (real) index of the pair that turns n times in L
        at = lambda n: d * math.log(L / (n * 2 * math.pi)) / (2 * math.log(float(theta)))  # noqa: E731
        lo, hi = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), d - 1)
        ramp = np.clip((np.arange(d // 2) - lo) / max(hi - lo, 1e-3), 0.0, 1.0)
        return w / f * ramp + w * (1.0 - ramp), float(scaling.get("attention",
                                                                  0.1 * math.log(f) + 1.0))
    low, high = float(scaling.get("low", 1.0)), float(scaling.get("high", 4.0))
    if not 0 < low < high:
        raise ValueError(f"expected 0 < low < high, got {low}, {high}")
    keep = np.clip((L * w / (2 * math.pi) - low) / (high - low), 0.0, 1.0)
    return (1.0 - keep) * w / f + keep * w, 1.0


class Rotary:
    """The plan of a model's rotary positions: layout, rotated part and frequencies (float64 on
    the device)."""

    def __init__(self, head_dim, theta=1e6, rotary_dim=None, layout="half", scaling=None,
                 device=None):
        self.head_dim = int(head_dim)
        self.rotary_dim = self.head_dim if rotary_dim is None else int(rotary_dim)
        if not 0 < self.rotary_dim <= self.head_dim or self.rotary_dim % 2:
            raise ValueError(f"rotary_dim {self.rotary_dim} must be even, in (0, "
                             f"{self.head_dim}]")
        if layout not in ("half", "interleaved"):
            raise ValueError(f"layout must be 'half' or 'interleaved', got {layout!r}")
        if not (float(theta) > 1.0 and math.isfinite(float(theta))):
            raise ValueError(f"theta must be a finite number > 1, got {theta}")
        self.layout = layout
        self.freqs, self.factor = frequencies(self.rotary_dim, theta, scaling)
        self.turns = torch.from_numpy(self.freqs / (2 * math.pi)).to(device or _lib.device())

    def _side(self, x, T, dtype, dev, what):
        """Strides of tokens and heads, and the heads, of x [T, heads, head_dim]."""
        shape = x.shape
        if len(shape) != 3 or x.dtype != dtype or shape[2] != self.head_dim or shape[0] != T:
            raise ValueError(f"{what} must be {dtype} [{T}, heads, {self.head_dim}], got "
                             f"{x.dtype} {tuple(shape)}")
        if shape[1] > MAX_HEADS:
            raise ValueError(f"{what} has more than {MAX_HEADS} heads")
        same_device(x, what, dev)
        st, sh, se = x.stride()
        if se != 1 and self.head_dim > 1:
            raise ValueError(f"{what}: the elements of a head must be contiguous")
        return st, sh, shape[1]

    def _out_side(self, o, x, T, dtype, dev, what):
        st, sh, n = self._side(o, T, dtype, dev, what)
        if n != x.shape[1]:
            raise ValueError(f"{what} must be {tuple(x.shape)}, got {tuple(o.shape)}")
        return st, sh

    @staticmethod
    def _outputs(q, k, qo, ko):
        """Refuses outputs that a thread could write before another one has read its input: each
        lies on its own input, or apart from both inputs, and apart from the other output."""
        if k is None or not k.numel():
            k = ko = None
        # the usual layouts are settled by a few comparisons (every call with `out` comes here)
        bq, bk, bqo, bko = box(q), box(k), box(qo), box(ko)
        if bqo[4] and bko[4] and boxes_apart(bqo, bko) and boxes_apart(bqo, bk) and \
                boxes_apart(bko, bq) and (same_rows(qo, q) or boxes_apart(bqo, bq)) and \
                (k is None or same_rows(ko, k) or boxes_apart(bko, bk)):
            return
        ins = [("q", q, runs(q))] + ([] if k is None else [("k", k, runs(k))])
        outs = []
        for (name, x, _), o in zip(ins, (qo, ko)):
            to, what = runs(o), name + "_out"
            if repeats(to):
                raise ValueError(f"{what} must not repeat its elements")
            for other, _, rows in ins:
                if not (other == name and same_rows(o, x)) and meet(to, rows):
                    raise ValueError(f"{what} overlaps {other} without being the same rows")
            outs.append(to)
        if len(outs) == 2 and meet(*outs):
            raise ValueError("k_out overlaps q_out")

    def _turn(self, q, k, positions, out, inverse):
        code = DTYPES.get(q.dtype)
        if q.dim() != 3 or code is None:
            raise ValueError(f"q must be a bf16, float16 or float32 [T, heads, {self.head_dim}] "
                             f"tensor, got {q.dtype} {tuple(q.shape)}")
        dev = on_device(q, "q")
        T, dt, hd = q.shape[0], q.dtype, self.head_dim
        q_t, q_h, nq = self._side(q, T, dt, dev, "q")
        if not nq and T:
            raise ValueError("q must have at least one head")
        k_t, k_h, nk = (0, 0, 0) if k is None else self._side(k, T, dt, dev, "k")
        wide = positions.dtype is torch.int64
        if not wide and positions.dtype is not torch.int32 or positions.shape != (T,):
            raise ValueError(f"positions must be int32 or int64 [{T}], got {positions.dtype} "
                             f"{tuple(positions.shape)}")
        same_device(positions, "positions", dev)
        same_device(self.turns, "the plan", dev)
        if not positions.is_contiguous():
            positions = positions.contiguous()
        if out is None:
            qo, qo_t, qo_h = q.new_empty((T, nq, hd)), nq * hd, hd
            ko, ko_t, ko_h = None if k is None else k.new_empty((T, nk, hd)), nk * hd, hd
        else:
            qo, ko = out
            if qo is None or (ko is None) != (k is None):
                raise ValueError("out must be (q_out, k_out), k_out None without k")
            qo_t, qo_h = self._out_side(qo, q, T, dt, dev, "q_out")
            ko_t, ko_h = (0, 0) if k is None else self._out_side(ko, k, T, dt, dev, "k_out")
            if T:
                self._outputs(q, k, qo, ko)
        if T:
            _lib.call("gsq_rope", q.data_ptr(), q_t, q_h, nq, k.data_ptr() if nk else None, k_t,
                      k_h, nk, T, hd, self.rotary_dim, self.layout == "interleaved", code, positions.data_ptr(),
                      wide, self.turns.data_ptr(), self.factor, inverse, qo.data_ptr(), qo_t, qo_h,
                      ko.data_ptr() if nk else None, ko_t, ko_h, stream_of(dev))
        return qo, ko

    def __call__(self, q, k, positions, out=None):
        """q [T, heads, head_dim], k [T, kv heads, head_dim] (or None) of one type (bf16, float16,
        float32), rotated by the tokens' positions int32 / int64 [T]: (q', k'), new contiguous
        tensors or out = (q_out, k_out). Tokens and heads may be strided (views of a packed
        q | k | v buffer, head-major buffers transposed). In place with out = (q, k); any other
        overlap of an output with an input or with the other output is refused."""
        return self._turn(q, k, positions, out, False)

    def vjp(self, dq, dk, positions, out=None):
        """The cotangents of q and k from those of q' and k': the rotation by the opposite angles
        (same arguments as the forward)."""
        return self._turn(dq, dk, positions, out, True)
