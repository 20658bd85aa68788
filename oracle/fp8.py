"""Restatement of the e4m3 block format and its products in float64 numpy (test infrastructure)."""
import numpy as np

BLOCK = 128


def e4m3(v):
    """v (float64) to the nearest e4m3 value, ties to even: 3 fraction bits, least exponent -6,
    magnitudes up to 448 (larger ones saturate), NaN kept."""
    v = np.asarray(v, np.float64)
    _, e = np.frexp(np.where(np.isfinite(v), v, 0.0))
    step = np.ldexp(1.0, np.maximum(e - 1, -6) - 3)
    q = np.clip(np.rint(np.where(np.isfinite(v), v, 0.0) / step) * step, -448.0, 448.0)
    return np.where(np.isnan(v), np.nan, np.where(np.isinf(v), np.sign(v) * 448.0, q))


def _encode(b, axis):
    """(values of the codes, scale) of float32 blocks along the axes given."""
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        a = np.maximum(np.max(np.abs(b), axis=axis, keepdims=True), np.float32(2.0 ** -100))
        r = np.float32(448.0) / a
        return e4m3((b * r).astype(np.float32)), a / np.float32(448.0)


def quantize_rows(x):
    """x [R, C] float32 -> (codes' values [R, C], scales [R, blocks])."""
    x = np.asarray(x, np.float32)
    R, C = x.shape
    nb = -(-C // BLOCK)
    p = np.zeros((R, nb * BLOCK), np.float32)
    p[:, :C] = x
    q, s = _encode(p.reshape(R, nb, BLOCK), 2)
    return q.reshape(R, -1)[:, :C], s.reshape(R, nb)


def quantize_blocks(w):
    """w [N, K] float32 -> (codes' values [N, K], scales [N blocks, K blocks])."""
    w = np.asarray(w, np.float32)
    N, K = w.shape
    nb, kb = -(-N // BLOCK), -(-K // BLOCK)
    p = np.zeros((nb * BLOCK, kb * BLOCK), np.float32)
    p[:N, :K] = w
    q, s = _encode(p.reshape(nb, BLOCK, kb, BLOCK), (1, 3))
    return q.reshape(nb * BLOCK, -1)[:N, :K], s.reshape(nb, kb)


def rows_value(q, s):
    return q * np.repeat(s.astype(np.float64), BLOCK, 1)[:, :q.shape[1]]


def blocks_value(q, s):
    return q * np.repeat(np.repeat(s.astype(np.float64), BLOCK, 0)[:q.shape[0]], BLOCK,
                         1)[:, :q.shape[1]]


def linear(x, qw, sw):
    """(y, the sum of the products' magnitudes) of x [M, K] float32 and a weight's codes."""
    xv, wv = rows_value(*quantize_rows(x)), blocks_value(qw, sw)
    return xv @ wv.T, np.abs(xv) @ np.abs(wv).T


def vjp(x, dy, qw, sw):
    """(dx, its magnitudes, dw, its magnitudes)."""
    dv, wv = rows_value(*quantize_rows(dy)), blocks_value(qw, sw)
    dt, xt = rows_value(*quantize_rows(dy.T)), rows_value(*quantize_rows(x.T))
    return dv @ wv, np.abs(dv) @ np.abs(wv), dt @ xt.T, np.abs(dt) @ np.abs(xt).T
