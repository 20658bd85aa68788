"""Restatement of the rotary positions and of the residual norms in float64 (test infrastructure)."""
import numpy as np


def rotate(x, positions, freqs, rotary_dim, layout, factor=1.0, inverse=False):
    """x [T, heads, hd] float64 turned pair by pair (a loop over pairs, complex products)."""
    x = np.asarray(x, np.float64)
    out = x.copy()
    t = np.asarray(positions, np.float64)[:, None]
    for j in range(rotary_dim // 2):
        a, b = (j, j + rotary_dim // 2) if layout == "half" else (2 * j, 2 * j + 1)
        z = (x[..., a] + 1j * x[..., b]) * factor * np.exp((-1j if inverse else 1j) * t * freqs[j])
        out[..., a], out[..., b] = z.real, z.imag
    return out


def _rows(gate, T):
    return 1.0 if gate is None else np.repeat(np.atleast_2d(gate),
                                              T // np.atleast_2d(gate).shape[0], 0)


def residual_norm(h, y, w_post, w_pre, gate=None, scale=1.0, eps=1e-6, offset=0.0):
    """(h', x, r1, r2, n): float64 rows."""
    T = h.shape[0]
    r1 = np.ones((T, 1)) if w_post is None else 1 / np.sqrt((y * y).mean(1, keepdims=True) + eps)
    n = y if w_post is None else y * r1 * (w_post + offset)
    h2 = h + scale * _rows(gate, T) * n
    r2 = np.ones((T, 1)) if w_pre is None else 1 / np.sqrt((h2 * h2).mean(1, keepdims=True) + eps)
    x = None if w_pre is None else h2 * r2 * (w_pre + offset)
    return h2, x, r1, r2, n


def residual_norm_vjp(h, y, w_post, w_pre, dh, dx, gate=None, scale=1.0, eps=1e-6, offset=0.0):
    """({name: gradient}, {name: sum of the magnitudes it is made of})."""
    T, H = h.shape
    h2, _, r1, r2, n = residual_norm(h, y, w_post, w_pre, gate, scale, eps, offset)
    g = _rows(gate, T)
    d = np.zeros_like(h) if dh is None else dh
    dm = np.abs(d)
    out, mag = {}, {}
    if w_pre is not None:
        hn, u = h2 * r2, dx * (w_pre + offset)
        d = d + r2 * (u - hn * (u * hn).mean(1, keepdims=True))
        dm = dm + r2 * (np.abs(u) + np.abs(hn) * np.abs(u * hn).mean(1, keepdims=True))
        # h' itself carries the rounding of its two summands, which may cancel
        hm = (np.abs(h) + np.abs(scale * g * n)) * r2
        dm = dm + r2 * hm * np.abs(u * hn).mean(1, keepdims=True) \
            + r2 * np.abs(hn) * (np.abs(u) * hm).mean(1, keepdims=True)
        out["dw_pre"], mag["dw_pre"] = (dx * hn).sum(0), (np.abs(dx) * (np.abs(hn) + hm)).sum(0)
    out["dh"], mag["dh"] = d, dm
    m, mm = scale * g * d, np.abs(scale * g) * dm
    if gate is not None:
        G = np.atleast_2d(gate).shape[0]
        out["dgate"] = (scale * d * n).reshape(G, -1, H).sum(1).reshape(np.shape(gate))
        mag["dgate"] = (abs(scale) * dm * np.abs(n)).reshape(G, -1, H).sum(1).reshape(
            np.shape(gate))
    if w_post is None:
        out["dy"], mag["dy"] = m, mm
        return out, mag
    yn, a = y * r1, w_post + offset
    v, vm = m * a, mm * np.abs(a)
    out["dy"] = r1 * (v - yn * (v * yn).mean(1, keepdims=True))
    mag["dy"] = r1 * (vm + np.abs(yn) * (vm * np.abs(yn)).mean(1, keepdims=True))
    out["dw_post"], mag["dw_post"] = (m * yn).sum(0), (mm * np.abs(yn)).sum(0)
    return out, mag
