"""The oracles of the 8-bit linear, the rotary positions and the residual norms (known values,
gradients against differences), and the refusals of the operators: host checks and the C ABI's
checks, which need no GPU."""
import ctypes as C

import numpy as np
import pytest
import torch

from gsq_rco_mlx_b200 import _lib
from gsq_rco_mlx_b200.common import fp8, norm, rotary
from oracle import blockops as ob
from oracle import fp8 as of

P = C.c_void_p(4096)   # 16-byte aligned, never dereferenced: every call below is refused first


def test_e4m3_rounding():
    """All 256 codes are fixed points, torch's own cast agrees, ties go to even."""
    codes = torch.arange(256, dtype=torch.int32).to(torch.uint8).view(torch.float8_e4m3fn)
    vals = codes.float().numpy().astype(np.float64)
    ok = np.isfinite(vals)
    assert ok.sum() == 254
    assert np.array_equal(of.e4m3(vals[ok]), vals[ok])
    x = np.concatenate([np.linspace(-460, 460, 100001), np.ldexp(1.0, np.arange(-14, 9)),
                        np.arange(-64, 65) * 2.0 ** -10]).astype(np.float32)
    t = torch.from_numpy(x).clamp(-448, 448).to(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(of.e4m3(x.astype(np.float64)), t)
    assert of.e4m3(np.array([17.0]))[0] == 16.0 and of.e4m3(np.array([19.0]))[0] == 20.0
    assert np.isnan(of.e4m3(np.array([np.nan])))[0]


def test_quantized_blocks_hold_their_bounds():
    """Half a step of e4m3 (2^-4 of the value) or of its least step (2^-10, times the scale)."""
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((7, 300)) * np.exp(3 * rng.standard_normal((7, 300)))).astype(
        np.float32)
    x[2, :128] = 0
    q, s = of.quantize_rows(x)
    v = of.rows_value(q, s)
    sc = np.repeat(s, 128, 1)[:, :300]
    # (the product by the reciprocal, and the scale, round by 2^-24 each: 2^-22 covers them)
    assert np.all(np.abs(v - x) <= np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** -10 * sc)
                  * (1 + 2.0 ** -18) + 2.0 ** -22 * np.abs(x))
    assert np.all(np.max(np.abs(q).reshape(7, -1)[:, :128], 1)[[0, 1, 3, 4, 5, 6]] == 448)
    assert np.all(v[2, :128] == 0)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotation_is_its_own_transpose_inverse(layout):
    rng = np.random.default_rng(1)
    q, u = rng.standard_normal((2, 5, 3, 10))
    pos = np.array([0, 1, -7, 100000, 3])
    w, f = rotary.frequencies(8, 1e4, {"type": "yarn", "factor": 4.0, "original": 64})
    r = ob.rotate(q, pos, w, 8, layout, f)
    # <R q, u> = <q, R^T u>
    np.testing.assert_allclose((r * u).sum(),
                               (q * ob.rotate(u, pos, w, 8, layout, f, inverse=True)).sum(),
                               rtol=1e-12)
    assert np.array_equal(r[..., 8:], q[..., 8:])
    np.testing.assert_allclose(np.linalg.norm(r[..., :8]), f * np.linalg.norm(q[..., :8]))


def test_frequencies():
    w, f = rotary.frequencies(64, 1e6)
    np.testing.assert_allclose(w, 1e6 ** (-np.arange(32) / 32), rtol=1e-15)
    assert f == 1.0
    assert np.array_equal(rotary.frequencies(64, 1e6, {"type": "linear", "factor": 4.0})[0], w / 4)
    n = rotary.frequencies(64, 1e6, {"type": "ntk", "factor": 4.0})[0]
    assert n[0] == 1.0 and n[-1] == pytest.approx(w[-1] / 4, rel=1e-12)
    y, fy = rotary.frequencies(64, 1e4, {"type": "yarn", "factor": 8.0, "original": 4096})
    w4 = rotary.frequencies(64, 1e4)[0]
    turns = 4096 * w4 / (2 * np.pi)
    assert np.all(y[turns > 40] == w4[turns > 40]) and np.allclose(y[turns < 0.7],
                                                                   w4[turns < 0.7] / 8)
    assert np.all(np.diff(y) < 0) and fy == pytest.approx(0.1 * np.log(8.0) + 1)
    b = rotary.frequencies(64, 1e4, {"type": "bands", "factor": 8.0, "original": 4096})[0]
    assert np.all(b[turns >= 4] == w4[turns >= 4]) and np.allclose(b[turns <= 1],
                                                                   w4[turns <= 1] / 8)
    for bad in ({"type": "other", "factor": 2.0}, {"type": "linear"},
                {"type": "linear", "factor": 0.5}, {"type": "linear", "factor": float("inf")},
                {"type": "yarn", "factor": 2.0}, {"type": "linear", "factor": 2.0, "low": 1},
                {"type": "bands", "factor": 2.0, "original": 64, "low": 4.0, "high": 1.0},
                {"type": "yarn", "factor": 2.0, "original": 64, "slow": 0.0}):
        with pytest.raises(ValueError):
            rotary.frequencies(64, 1e4, bad)


@pytest.mark.parametrize("post,pre,gates", [(True, True, 0), (True, True, 1), (True, True, 3),
                                            (False, True, 6), (True, False, 2)])
def test_norm_gradients_against_differences(post, pre, gates):
    """The oracle's gradients against central differences of its forward pass: step 1e-5, so the
    truncation is 1e-10 of third derivatives of order 1 and the rounding 1e-16 / 1e-5."""
    rng = np.random.default_rng(2)
    T, H = 6, 9
    v = {"h": rng.standard_normal((T, H)), "y": rng.standard_normal((T, H))}
    if post:
        v["w_post"] = rng.standard_normal(H)
    if pre:
        v["w_pre"] = rng.standard_normal(H)
    if gates:
        v["gate"] = rng.standard_normal((gates, H))
    dh = rng.standard_normal((T, H))
    dx = rng.standard_normal((T, H)) if pre else None

    def value(v):
        h2, x, *_ = ob.residual_norm(v["h"], v["y"], v.get("w_post"), v.get("w_pre"),
                                     v.get("gate"), 0.7, 1e-3, 1.0)
        return (h2 * dh).sum() + (0.0 if x is None else (x * dx).sum())

    g, _ = ob.residual_norm_vjp(v["h"], v["y"], v.get("w_post"), v.get("w_pre"), dh, dx,
                                v.get("gate"), 0.7, 1e-3, 1.0)
    for name in v:
        grad = g["d" + name]
        assert grad.shape == v[name].shape
        for i in np.ndindex(v[name].shape):
            up, dn = dict(v), dict(v)
            up[name], dn[name] = v[name].copy(), v[name].copy()
            up[name][i] += 1e-5
            dn[name][i] -= 1e-5
            assert grad[i] == pytest.approx((value(up) - value(dn)) / 2e-5, rel=1e-6, abs=1e-7)


def test_fp8_gradients_against_differences():
    """dx of y = q(x) W^T with the rounding counted as the identity is the gradient through W's
    values, dw that through the (column-quantized) x: both against differences of the bilinear
    form, which is exact up to rounding for any step."""
    rng = np.random.default_rng(3)
    x, dy = (rng.standard_normal(s).astype(np.float32) for s in ((150, 200), (150, 140)))
    qw, sw = of.quantize_blocks(rng.standard_normal((140, 200)).astype(np.float32))
    dx, _, dw, _ = of.vjp(x, dy, qw, sw)
    dv, wv = of.rows_value(*of.quantize_rows(dy)), of.blocks_value(qw, sw)
    dt, xt = of.rows_value(*of.quantize_rows(dy.T)).T, of.rows_value(*of.quantize_rows(x.T)).T
    for (i, k) in ((0, 0), (149, 199), (70, 130)):
        f = lambda e: ((x[i] + e * (np.arange(200) == k)) @ wv.T * dv[i]).sum()  # noqa: E731
        assert dx[i, k] == pytest.approx(f(1.0) - f(0.0), rel=1e-6, abs=1e-9)
    for (n, k) in ((0, 0), (139, 199), (128, 127)):
        f = lambda e: (xt @ (wv[n] + e * (np.arange(200) == k)) * dt[:, n]).sum()  # noqa: E731
        assert dw[n, k] == pytest.approx(f(1.0) - f(0.0), rel=1e-6, abs=1e-9)


def test_operators_refuse_host_tensors():
    x = torch.zeros(4, 64)
    with pytest.raises(ValueError):
        fp8.quantize_rows(x)
    with pytest.raises(ValueError):
        fp8.Fp8Linear.from_weight(x)
    with pytest.raises(ValueError):
        fp8.Fp8Linear(torch.zeros(4, 64, dtype=torch.float8_e4m3fn), torch.zeros(1, 1))
    with pytest.raises(ValueError):
        fp8.Fp8Linear(x, torch.zeros(1, 1))
    with pytest.raises(ValueError):
        norm.residual_norm(x, x, w_pre=torch.zeros(64))
    for kw in ({"rotary_dim": 3}, {"rotary_dim": 66}, {"rotary_dim": 0}, {"layout": "pairs"},
               {"theta": 1.0}, {"scaling": {"type": "linear", "factor": -1}}):
        with pytest.raises(ValueError):
            rotary.Rotary(64, device="cpu", **kw)
    r = rotary.Rotary(64, device="cpu")
    for q, k, pos in ((torch.zeros(4, 2, 64), None, torch.zeros(4, dtype=torch.int32)),
                      (torch.zeros(4, 64), None, torch.zeros(4, dtype=torch.int32)),
                      (torch.zeros(4, 2, 64, dtype=torch.float64), None,
                       torch.zeros(4, dtype=torch.int32))):
        with pytest.raises(ValueError):
            r(q, k, pos)


def _refused(fn, ok, bad, status=_lib.GSQ_EINVAL):
    for i, v in bad:
        args = list(ok)
        args[i] = v
        assert fn(*args) == status, (i, v)


def test_transposed_codes_are_not_made_during_a_capture(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    lin = fp8.Fp8Linear.__new__(fp8.Fp8Linear)
    lin.N, lin.K, lin._t = 16, 32, None
    lin.codes = torch.zeros(16, 32, dtype=torch.uint8).view(torch.float8_e4m3fn)
    with pytest.raises(RuntimeError, match="before it"):
        lin.codes_t()
    assert lin._t is None


def test_quantized_rows_are_no_input_of_the_gradient():
    """Refused with the reason, not with an error of a missing attribute."""
    lin = fp8.Fp8Linear.__new__(fp8.Fp8Linear)
    q = fp8.Fp8Tensor.empty(4, 32, torch.device("cpu"))
    with pytest.raises(ValueError, match="x must be dense"):
        lin.vjp(q, torch.zeros(4, 16))


def test_the_error_word_is_not_made_during_a_capture(monkeypatch):
    """Nor is one that is there asked for again."""
    from gsq_rco_mlx_b200 import gemm
    from gsq_rco_mlx_b200.common import operands
    dev = torch.device("cpu")
    monkeypatch.setattr(gemm, "_ERR", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="before"):
        operands.error_word(dev)
    assert not gemm._ERR
    word = gemm.err_flag(dev)
    assert operands.error_word(dev) is word


class _Waited:
    """A stream that notes whether the device's word could be had before its fill was waited for."""

    def __init__(self, words, dev, seen):
        self.words, self.dev, self.seen = words, dev, seen

    def synchronize(self):
        self.seen.append(self.dev in self.words)


def test_the_error_word_is_filled_before_it_can_be_had(monkeypatch):
    """Another stream's kernels read it: the fill is waited for before the word is kept."""
    from gsq_rco_mlx_b200 import gemm
    dev, seen, words = torch.device("cpu"), [], {}
    monkeypatch.setattr(gemm, "_ERR", words)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: _Waited(words, dev, seen))
    word = gemm.err_flag(dev)
    assert seen == [False] and words[dev] is word and int(word) == 0
    assert gemm.err_flag(dev) is word and seen == [False]


def test_an_error_word_made_in_a_capture_is_filled_by_the_next_eager_call(monkeypatch):
    """In a capture the fill only runs with the graph; kernels outside of it do not wait for that."""
    from gsq_rco_mlx_b200 import gemm
    dev, seen, words = torch.device("cpu"), [], {}
    monkeypatch.setattr(gemm, "_ERR", words)
    monkeypatch.setattr(gemm, "_UNFILLED", set())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: _Waited(words, dev, seen))
    word = gemm.err_flag(dev)
    assert gemm.err_flag(dev) is word and seen == []
    word.fill_(77)   # what lay there
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    assert gemm.err_flag(dev) is word and int(word) == 0 and len(seen) == 1
    word.fill_(3)    # an error from then on stays
    assert gemm.err_flag(dev) is word and int(word) == 3 and len(seen) == 1


def test_an_error_word_made_in_a_capture_is_known_as_that_from_the_first(monkeypatch):
    """Another host thread looks it up without the lock: it must not take it for a filled one."""
    from gsq_rco_mlx_b200 import gemm
    dev, unfilled, order = torch.device("cpu"), set(), []

    class Words(dict):
        def __setitem__(self, key, word):
            order.append(key in unfilled)
            super().__setitem__(key, word)

    monkeypatch.setattr(gemm, "_ERR", Words())
    monkeypatch.setattr(gemm, "_UNFILLED", unfilled)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    gemm.err_flag(dev)
    assert order == [True]


def test_outputs_over_inputs():
    """row_by_row against the elements themselves: it takes the same rows and every pair without a
    common element of one pitch or apart as a whole, and no pair with one."""
    from gsq_rco_mlx_b200.common.operands import row_by_row
    base = torch.zeros(256, dtype=torch.bfloat16)
    cell = torch.arange(256)
    for rows in (1, 2, 3):
        for cols in (1, 4):
            for lx in (4, 9):
                for lo in (4, 9):
                    for at in range(0, 41):
                        view = lambda t, ld, o: t[o:].as_strided((rows, cols), (ld, 1), o)  # noqa: E731
                        xs = set(view(cell, lx, 20).flatten().tolist())
                        os = set(view(cell, lo, at).flatten().tolist())
                        same = at == 20 and (lo == lx or rows == 1)
                        spans = max(os) < min(xs) or min(os) > max(xs)
                        args = (view(base, lo, at), lo, view(base, lx, 20), lx, "out", "h")
                        if same or not (os & xs) and (lo == lx or spans):
                            row_by_row(*args)
                        elif os & xs:
                            with pytest.raises(ValueError, match="overlaps h"):
                                row_by_row(*args)


def test_runs_that_meet():
    """meet and repeats against the elements themselves, over strided tensors of three dimensions
    in one buffer; settled by the extents where they lie as buffers of tokens and heads do."""
    from gsq_rco_mlx_b200.common import operands
    rng = np.random.default_rng(7)
    base = torch.zeros(4096, dtype=torch.float16)
    cell = torch.arange(4096)

    def some():
        T, n, hd = (int(rng.integers(1, 5)) for _ in range(3))
        st, sh = int(rng.integers(0, 40)), int(rng.integers(0, 40))
        return (T, n, hd), (st, sh, 1), int(rng.integers(0, 200))

    met = apart = again = 0
    for _ in range(3000):
        a, b = some(), some()
        if rng.random() < 0.5:   # two parts of one packed buffer, often
            b = (b[0], a[1], b[2])
        va, vb = (base.as_strided(*x) for x in (a, b))
        ea, eb = (cell.as_strided(*x).flatten().tolist() for x in (a, b))
        want = bool(set(ea) & set(eb))
        assert operands.meet(operands.runs(va), operands.runs(vb)) == want, (a, b)
        assert operands.repeats(operands.runs(va)) == (len(set(ea)) < len(ea)), a
        xa, xb = operands.box(va), operands.box(vb)
        assert not (want and operands.boxes_apart(xa, xb)), (a, b)
        assert not (xa[4] and len(set(ea)) < len(ea)), a
        if a[0] == b[0]:
            assert operands.same_rows(va, vb) == (ea == eb), (a, b)
        met, apart, again = met + want, apart + (not want), again + (len(set(ea)) < len(ea))
    assert min(met, apart, again) > 300
    # q | k | v rows, a buffer of heads, one of pairs of heads: no run is looked at by itself
    rows = base[:6 * 5 * 8].view(6, 5, 8)
    heads = base[:6 * 5 * 8].view(5, 6, 8).transpose(0, 1)
    for x in (rows, heads):
        for p, q in ((x[:, :3], x[:, 3:4]), (x[:, 4:], x[:, 0:4]), (x[:, 0::2], x[:, 1::2]),
                     (x[:2], x[2:]), (x[..., :4], x[..., 4:])):
            a, b = operands.runs(p), operands.runs(q)
            assert operands._surely_apart(a[1], a[2], b[1], b[2], b[0] - a[0])
    for x in (rows, heads):
        assert operands.boxes_apart(operands.box(x[:, :3]), operands.box(x[:, 3:4]))
    square = base[:4 * 4 * 8].view(4, 4, 8)
    assert not operands.same_rows(square, square.transpose(0, 1))


def test_outputs_over_other_tensors():
    """apart against the elements themselves, between types of different size."""
    from gsq_rco_mlx_b200.common.operands import apart
    rng = np.random.default_rng(8)
    buf = torch.zeros(512, dtype=torch.uint8)
    byte, seen = torch.arange(512), [0, 0]

    def some(dtype, n):
        r, c = (int(rng.integers(1, 5)) for _ in range(2))
        ld, at = int(rng.integers(c, 12)), int(rng.integers(0, 20))
        if rng.random() < 0.4:
            ld = c
        t = buf.view(dtype).as_strided((r, c), (ld, 1), at)
        return t, {int(v) for v in byte.as_strided((r, c, n), (ld * n, n, 1), at * n).flatten()}

    for _ in range(3000):
        (a, ea), (b, eb) = some(torch.float32, 4), some(torch.bfloat16, 2)
        seen[bool(ea & eb)] += 1
        if ea & eb:
            with pytest.raises(ValueError, match="a overlaps b"):
                apart(a, "a", b, "b")
        else:
            apart(a, "a", b, "b")
    assert min(seen) > 300
    apart(buf.view(torch.float32)[:0], "a", buf, "b")


def test_rotary_outputs_over_inputs():
    """On their own inputs, or apart from both and from one another; a buffer's elements once."""
    rot = rotary.Rotary(8, device="cpu")
    buf = torch.zeros(9, 6 * 8)
    part = lambda t0, t1, h0, h1: buf.view(9, 6, 8)[t0:t1, h0:h1]  # noqa: E731
    q, k = part(0, 4, 0, 2), part(0, 4, 2, 4)
    new = torch.zeros(4, 2, 8)
    hm = torch.zeros(2, 4, 8).transpose(0, 1)
    for out in ((q, k), (new, k), (q, new), (new, hm), (hm, new), (new, new.clone()),
                (part(4, 8, 0, 2), k), (part(0, 4, 4, 6), k), (q, part(5, 9, 2, 4))):
        rot._outputs(q, k, *out)
    rot._outputs(q, None, q, None)
    rot._outputs(q[:1], None, buf[:1, :16].view(1, 2, 8), None)   # (one token: its stride is none)
    slide = lambda t, d: t.as_strided(t.shape, t.stride(), t.storage_offset() + d)  # noqa: E731
    for out, match in (((part(1, 5, 0, 2), k), "overlaps q"), ((k, q), "overlaps"),
                       ((slide(q, 1), new), "overlaps"), ((slide(q, 8), new), "overlaps"),
                       ((new, part(3, 7, 0, 2)), "overlaps q"), ((part(0, 4, 2, 4), new), "overlaps k"),
                       ((new, new), "overlaps"), ((q[:, :1].expand(4, 2, 8), new), "repeat"), ((new, slide(new, 0)), "overlaps"),
                       ((buf.view(-1)[:64].view(4, 2, 8), new), "overlaps q"),
                       ((torch.zeros(64).as_strided((4, 2, 8), (1, 8, 1)), k), "repeat"),
                       ((torch.zeros(64).as_strided((4, 2, 8), (16, 4, 1)), k), "repeat")):
        with pytest.raises(ValueError, match=match):
            rot._outputs(q, k, *out)
    square = torch.zeros(4, 4, 8)
    with pytest.raises(ValueError, match="overlaps q"):
        rot._outputs(square, None, square.transpose(0, 1), None)
    with pytest.raises(ValueError, match="overlaps"):
        rot._outputs(q, q, q, q)   # one buffer twice: it would be turned twice


def test_sizes_past_32_bit_counts_are_refused():
    """Not cut to their low 32 bits (2^32 + 4 rows are not four), nor run with counts that a grid's
    step would overflow."""
    from gsq_rco_mlx_b200.common.operands import matrix
    cell = torch.zeros(1, 1, dtype=torch.bfloat16)
    code = cell.to(torch.float8_e4m3fn)
    for n in ((1 << 30) + 1, (1 << 32) + 4):
        for shape in ((n, 1), (1, n)):
            with pytest.raises(ValueError, match="more than"):
                matrix(cell.expand(*shape), "x")
            with pytest.raises(ValueError, match="more than"):
                fp8.Fp8Tensor(code.expand(*shape), torch.zeros(1, 1))
            with pytest.raises(ValueError, match="more than"):
                fp8.Fp8Linear(code.expand(*shape), torch.zeros(1, 1))
    rot = rotary.Rotary(2, device="cpu")
    with pytest.raises(ValueError, match="heads"):
        rot._side(cell.expand(1, (1 << 32) + 4, 2), 1, torch.bfloat16, -1, "q")
    lib, n = _lib.load(), (1 << 30) + 1
    assert lib.gsq_fp8_quant(P, 0, n, 1, 1, P, 16, P, n, None, 0, None, 0, None) == _lib.GSQ_EINVAL
    assert lib.gsq_fp8_gemm(n, 1, 1, P, 16, P, n, P, 16, P, 0, 1, 1, P, 0, 1, 0, P,
                            None) == _lib.GSQ_EINVAL
    assert lib.gsq_fp8_dequant(P, 16, P, 1, n, 1, P, 0, 1, None) == _lib.GSQ_EINVAL
    assert lib.gsq_fp8_linear(P, 0, n, 1, 1, P, 16, P, 1, 1, P, 0, 1, P, 1 << 40, P,
                              None) == _lib.GSQ_EINVAL
    assert lib.gsq_fp8_linear_vjp(P, 0, n, 1, 1, P, 0, 1, 1, P, 16, P, 1, P, 1, P, 1, 0, P, 1 << 40,
                                  P, None) == _lib.GSQ_EINVAL
    assert lib.gsq_residual_norm(P, 1, P, 1, P, P, None, 0, n, 1, 0, 1.0, 1e-6, 0.0, P, 1, P, 1,
                                 None, 0, None, 0, P, None) == _lib.GSQ_EINVAL
    size = C.c_int64()
    assert lib.gsq_residual_norm_bwd_workspace(n, 1, 0, 0, C.byref(size)) == _lib.GSQ_EINVAL
    assert lib.gsq_residual_norm_bwd(P, 1, P, 1, P, P, None, 0, P, P, 1, P, 1, n, 1, 0, 1.0, 0.0, P,
                                     1, P, 1, P, P, None, P, 1 << 40, P, None) == _lib.GSQ_EINVAL


def test_fp8_entry_points_refuse_bad_arguments():
    lib = _lib.load()
    odd = C.c_void_p(4097)
    _refused(lib.gsq_fp8_quant,
             [P, 0, 5, 200, 200, P, 208, P, 5, P, 16, P, 200, None],
             [(0, None), (1, 3), (1, -1), (2, 0), (3, 0), (4, 199), (6, 200), (6, 192), (7, None),
              (8, 4), (5, odd), (9, odd), (10, 5), (11, None), (12, 199), (0, odd)])
    assert lib.gsq_fp8_quant(P, 0, 5, 200, 200, None, 0, None, 0, None, 0, None, 0,
                             None) == _lib.GSQ_EINVAL
    _refused(lib.gsq_fp8_quant_blocks, [P, 0, 5, 200, 200, P, 208, P, 2, None],
             [(0, None), (1, 5), (2, 0), (3, 0), (4, 10), (5, None), (6, 200), (7, None), (8, 1)])
    _refused(lib.gsq_fp8_dequant, [P, 208, P, 2, 5, 200, P, 0, 200, None],
             [(0, None), (1, 200), (2, None), (3, 1), (4, 0), (5, 0), (6, None), (7, 3), (8, 199)])
    gemm = [8, 16, 200, P, 208, P, 8, P, 208, P, 0, 2, 1, P, 0, 16, 0, P, None]
    _refused(lib.gsq_fp8_gemm, gemm,
             [(0, 0), (1, 0), (2, 0), (3, None), (3, odd), (4, 200), (4, 192), (5, None), (6, 7),
              (7, None), (8, 200), (9, None), (11, -1), (13, None), (13, odd), (14, 3), (15, 15),
              (16, 1), (17, None)])
    rows = list(gemm)
    rows[10], rows[12] = 1, 15   # a scale per row needs its 16 rows in every block
    assert lib.gsq_fp8_gemm(*rows) == _lib.GSQ_EINVAL
    _refused(lib.gsq_fp8_linear, [P, 0, 8, 200, 200, P, 208, P, 2, 16, P, 0, 16, P, 8 * 216, P, None],
             [(0, None), (2, 0), (5, None), (6, 200), (8, 1), (9, 0), (10, None), (13, None),
              (13, odd), (14, 8 * 216 - 1), (15, None)])


def _tile(M, N, rows=0, accumulate=0, wide=1, sms=148):
    r, c = C.c_int(), C.c_int()
    assert _lib.load().gsq_fp8_gemm_tile(M, N, rows, accumulate, sms, wide, C.byref(r),
                                         C.byref(c)) == _lib.GSQ_OK
    return r.value, c.value


def test_fp8_product_tiles():
    """Few rows by themselves (not where a scale per row of both sides or a sum into the output is
    asked for), else by the rounds of the busiest multiprocessor; every tile is some size's."""
    assert [_tile(m, 4096) for m in (1, 16, 17, 32, 33, 64)] == \
        [(16, 128)] * 2 + [(32, 128)] * 2 + [(64, 128)] * 2
    assert _tile(64, 4096, rows=1)[0] >= 128 and _tile(64, 4096, accumulate=1)[0] >= 128
    assert _tile(16384, 4864) == (256, 256) and _tile(4864, 4864, rows=1) == (256, 256)
    assert _tile(600, 9000) == (256, 256) and _tile(600, 9000, rows=1) == (128, 128)
    assert _tile(100, 19000) == (128, 128) and _tile(100, 19000, rows=1) == (128, 128)
    lib, r, c = _lib.load(), C.c_int(), C.c_int()
    for bad in ((0, 1, 148), (1, 0, 148), ((1 << 30) + 1, 1, 148), (1, 1, 0)):
        assert lib.gsq_fp8_gemm_tile(bad[0], bad[1], 0, 0, bad[2], 1, C.byref(r),
                                     C.byref(c)) == _lib.GSQ_EINVAL
    assert lib.gsq_fp8_gemm_tile(1, 1, 0, 0, 148, 1, None, C.byref(c)) == _lib.GSQ_EINVAL


def test_fp8_product_without_the_wide_kernel():
    """A build whose wide kernel has another register count than its split needs takes the narrow
    tile, and the others stay."""
    sizes = [(m, n, s) for m in (65, 129, 300, 2047, 8191, 16384, 1 << 20, 1 << 30)
             for n in (1, 896, 4864, 19000, 1 << 30) for s in (0, 1)]
    for m, n, s in sizes:
        usual, narrow = _tile(m, n, s), _tile(m, n, s, wide=0)
        assert narrow == (128, 128)
        assert narrow == usual or usual == (256, 256)
    assert any(_tile(m, n, s) == (256, 256) for m, n, s in sizes)


def test_fp8_vjp_entry_point_refuses_bad_arguments():
    lib = _lib.load()
    need = 8 * 16 + (16 + 200) * 16 + 4 * (8 * 1 + (16 + 200) * 1)
    ok = [P, 0, 8, 200, 200, P, 0, 16, 16, P, 16, P, 2, P, 200, P, 200, 0, P, need, P, None]
    _refused(lib.gsq_fp8_linear_vjp, ok,
             [(0, None), (1, 3), (2, 0), (3, 0), (4, 199), (5, None), (6, -1), (7, 0), (8, 15),
              (9, None), (10, 15), (11, None), (12, 1), (13, None), (14, 199), (15, None),
              (16, 199), (18, None), (18, C.c_void_p(4100)), (19, need - 1), (20, None)])


def test_entry_points_refuse_pointers_off_their_type():
    """Scales, statistics, parameters and gradients that do not lie on their own size would be a
    misaligned access of the kernels."""
    lib, odd, two = _lib.load(), C.c_void_p(4097), C.c_void_p(4098)
    _refused(lib.gsq_fp8_quant, [P, 0, 5, 200, 200, P, 208, P, 5, P, 16, P, 200, None],
             [(7, two), (11, two)])
    _refused(lib.gsq_fp8_quant_blocks, [P, 0, 5, 200, 200, P, 208, P, 2, None], [(7, two)])
    _refused(lib.gsq_fp8_dequant, [P, 208, P, 2, 5, 200, P, 0, 200, None], [(2, two)])
    _refused(lib.gsq_fp8_gemm, [8, 16, 200, P, 208, P, 8, P, 208, P, 0, 2, 1, P, 0, 16, 0, P, None],
             [(5, two), (9, two), (17, two)])
    _refused(lib.gsq_fp8_linear, [P, 0, 8, 200, 200, P, 208, P, 2, 16, P, 0, 16, P, 8 * 216, P, None],
             [(7, two), (15, two)])
    need = 8 * 16 + (16 + 200) * 16 + 4 * (8 * 1 + (16 + 200) * 1)
    _refused(lib.gsq_fp8_linear_vjp,
             [P, 0, 8, 200, 200, P, 0, 16, 16, P, 16, P, 2, P, 200, P, 200, 0, P, need, P, None],
             [(11, two), (15, two), (20, two)])
    _refused(lib.gsq_residual_norm,
             [P, 64, P, 64, P, P, P, 2, 4, 64, 0, 1.0, 1e-6, 0.0, P, 64, P, 64, None, 0, None, 0, P,
              None], [(4, odd), (5, odd), (6, odd), (22, two)])
    _refused(lib.gsq_residual_norm,
             [P, 64, P, 64, P, P, P, 2, 4, 64, 2, 1.0, 1e-6, 0.0, P, 64, None, 0, P, 64, P, 4, P,
              None], [(4, two), (5, two), (6, two), (20, two)])
    _refused(lib.gsq_residual_norm_bwd,
             [P, 64, P, 64, P, P, P, 2, P, P, 64, P, 64, 4, 64, 0, 1.0, 0.0, P, 64, P, 64, P, P, P,
              P, 1 << 40, P, None],
             [(4, odd), (5, odd), (6, odd), (8, two), (22, two), (23, two), (24, two), (27, two)])


def test_rope_entry_point_refuses_bad_arguments():
    lib = _lib.load()
    ok = [P, 128, 64, 2, P, 128, 64, 1, 4, 64, 32, 0, 0, P, 0, P, 1.0, 0, P, 128, 64, P, 64, 64, None]
    _refused(lib.gsq_rope, ok,
             [(0, None), (3, 0), (4, None), (7, -1), (8, 0), (9, 0), (10, 0), (10, 31), (10, 66),
              (12, 3), (13, None), (13, C.c_void_p(4098)), (15, None), (15, C.c_void_p(4100)),
              (18, None), (21, None), (0, C.c_void_p(4097))])


def test_norm_entry_points_refuse_bad_arguments():
    lib = _lib.load()
    fwd = [P, 64, P, 64, P, P, P, 2, 4, 64, 0, 1.0, 1e-6, 0.0, P, 64, P, 64, None, 0, None, 0, P, None]
    _refused(lib.gsq_residual_norm, fwd,
             [(0, None), (1, 63), (2, None), (3, 63), (5, None), (7, 3), (7, 0), (8, 0), (9, 0),
              (10, 3), (15, 63), (16, None), (17, 63), (18, P), (22, None), (0, C.c_void_p(4097))])
    q = list(fwd)
    q[16], q[18], q[19], q[20], q[21] = None, P, 64, P, 4
    _refused(lib.gsq_residual_norm, q, [(19, 65), (19, 48), (20, None), (21, 3),
                                        (18, C.c_void_p(4104))])
    wide = list(fwd)
    for i in (1, 3, 9, 15, 17):
        wide[i] = 32769
    assert lib.gsq_residual_norm(*wide) == _lib.GSQ_ENOTSUP
    n = C.c_int64()
    for bad in ((0, 64, 0, 0), (4, 0, 0, 0), (4, 64, 0, 3), (4, 64, 0, -1), (4, 64, 3, 0)):
        assert lib.gsq_residual_norm_bwd_workspace(*bad, C.byref(n)) == _lib.GSQ_EINVAL
    assert lib.gsq_residual_norm_bwd_workspace(4, 64, 0, 0, None) == _lib.GSQ_EINVAL
    bwd = [P, 64, P, 64, P, P, P, 2, P, P, 64, P, 64, 4, 64, 0, 1.0, 0.0, P, 64, P, 64, P, P, P, P,
           1 << 40, P, None]
    _refused(lib.gsq_residual_norm_bwd, bwd,
             [(0, None), (1, 63), (2, None), (6, None), (7, 3), (8, None), (10, 63), (11, None),
              (12, 63), (13, 0), (14, 0), (15, 3), (18, None), (20, None), (22, None), (23, None),
              (24, None), (25, None), (26, 16), (27, None)])
    none = list(bwd)
    none[5], none[9], none[11], none[23] = None, None, None, None   # neither cotangent
    assert lib.gsq_residual_norm_bwd(*none) == _lib.GSQ_EINVAL
