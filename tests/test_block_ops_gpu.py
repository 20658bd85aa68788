"""The 8-bit linear, the rotary positions and the residual norms on the GPU against the float64
oracles, at the sizes, layouts and values where they can go wrong. The tolerances count roundings:
u = 2^-24 of float32, half a step of the output's type, and the number of float32 operations
between input and output, each applied to the magnitudes that the operation adds up."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from oracle import blockops as ob
from oracle import fp8 as of

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def half(dtype):
    """Half a step of the type, relative (float32 outputs round by U)."""
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half the least step of the type (its denormals)."""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


def f64(t):
    return t.detach().double().cpu().numpy()


def f32(t):
    return t.detach().float().cpu().numpy()


def rnd(shape, seed, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(*shape, generator=g)).to(dtype).cuda()


def near(got, want, tol, what=""):
    d = np.abs(got - want) - tol
    assert np.all(d <= 0), f"{what}: off by {d.max()} more than allowed at {np.argmax(d)}"


# ------------------------------------------------------------------------------ 8-bit linear ---
def _err_ok():
    from gsq_rco_mlx_b200.gemm import check_err
    torch.cuda.synchronize()
    check_err(torch.device("cuda", torch.cuda.current_device()))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("R,C", [(1, 1), (1, 128), (3, 129), (130, 127), (17, 896), (257, 1000),
                                 (128, 256), (5, 4864)])
def test_quantized_codes_are_the_oracles(R, C, dtype):
    """Rows, weights (128 x 128) and columns: codes and scales bit for bit."""
    from gsq_rco_mlx_b200 import _lib
    from gsq_rco_mlx_b200.common.fp8 import Fp8Linear, quantize_rows
    x = rnd((R, C), R + C, DT[dtype]) * torch.exp(2 * rnd((R, 1), 1)).to(DT[dtype])
    x[0, :100] = 0
    q = quantize_rows(x)
    qo, so = of.quantize_rows(f32(x))
    assert np.array_equal(f32(q.codes), qo) and np.array_equal(f32(q.scales), so)
    lin = Fp8Linear.from_weight(x)
    qo, so = of.quantize_blocks(f32(x))
    assert np.array_equal(f32(lin.codes), qo) and np.array_equal(f32(lin.scales), so)
    assert np.array_equal(f32(lin.codes_t()), qo.T)
    ld, rb = -(-R // 16) * 16, -(-R // 128)
    codes_t = torch.zeros(C, ld, device="cuda", dtype=torch.uint8)
    scales_t = torch.zeros(rb, C, device="cuda")
    _lib.call("gsq_fp8_quant", x.data_ptr(), list(DT).index(dtype), R, C, C, None, 0, None, 0,
              codes_t.data_ptr(), ld, scales_t.data_ptr(), C, _lib.stream_ptr())
    qo, so = of.quantize_rows(f32(x).T)
    assert np.array_equal(f32(codes_t.view(torch.float8_e4m3fn)[:, :R]), qo)
    assert np.array_equal(f32(scales_t), so.T)
    out = torch.empty(R, C, device="cuda", dtype=DT[dtype])
    lin.dequant(out)
    v = of.blocks_value(*of.quantize_blocks(f32(x)))
    near(f64(out), v, (half(DT[dtype]) + U) * np.abs(v) + tiny(DT[dtype]))


def _tol_gemm(mag, K, dtype, ref):
    """A block's 128 products are exact; their float32 sum on the tensor cores may truncate, one
    step (2 u) for each of 128 additions; the scales' product, the multiply by it (two with a
    scale per row of both sides) and the addition over blocks round by u each."""
    return (256 + 3 + -(-K // 128)) * U * mag + half(dtype) * np.abs(ref) * (1 + 1e-6) + tiny(dtype)


SHAPES = [(1, 1, 1), (1, 896, 1152), (2, 130, 257), (8, 128, 128), (16, 4864, 896), (17, 1000, 64),
          (64, 896, 4864), (65, 257, 333), (129, 128, 1), (300, 129, 1000), (1000, 896, 900),
          (2047, 64, 4864)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_fp8_linear(M, K, N, dtype):
    from gsq_rco_mlx_b200.common.fp8 import Fp8Linear, quantize_rows
    lin = Fp8Linear.from_weight(rnd((N, K), 1, scale=0.05))
    x = rnd((M, K), 2, DT[dtype])
    y = lin(x)
    y32 = lin(x, y_f32=True)
    yq = lin(quantize_rows(x))
    _err_ok()
    ref, mag = of.linear(f32(x), f32(lin.codes), f32(lin.scales))
    assert y.dtype == DT[dtype] and y32.dtype == torch.float32 and yq.dtype == torch.bfloat16
    near(f64(y), ref, _tol_gemm(mag, K, DT[dtype], ref))
    near(f64(y32), ref, _tol_gemm(mag, K, torch.float32, ref))
    near(f64(yq), ref, _tol_gemm(mag, K, torch.bfloat16, ref))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("M,K,N", SHAPES[1:])
def test_fp8_vjp(M, K, N, dtype):
    from gsq_rco_mlx_b200.common.fp8 import Fp8Linear
    lin = Fp8Linear.from_weight(rnd((N, K), 3, scale=0.05), transposed=M % 2 == 0)
    x, dy = rnd((M, K), 4, DT[dtype]), rnd((M, N), 5, DT[dtype], 0.01)
    dx, dw = lin.vjp(x, dy)
    base = rnd((N, K), 6)
    acc = base.clone()
    lin.vjp(x, dy, dw=acc, accumulate=True)
    _err_ok()
    rx, mx, rw, mw = of.vjp(f32(x), f32(dy), f32(lin.codes), f32(lin.scales))
    near(f64(dx), rx, _tol_gemm(mx, N, DT[dtype], rx), "dx")
    near(f64(dw), rw, _tol_gemm(mw, M, torch.float32, rw), "dw")
    near(f64(acc), rw + f64(base), _tol_gemm(mw, M, torch.float32, rw)
         + U * np.abs(rw + f64(base)), "dw added")


def test_fp8_long_and_wide():
    """More k-blocks than a CTA of the few-row product stages scales for at a time, with no split
    of k; and the widest tiles with a scale per row of both sides (dW of a square weight)."""
    from gsq_rco_mlx_b200.common.fp8 import Fp8Linear
    lin = Fp8Linear.from_weight(rnd((19000, 2600), 1, torch.bfloat16, 0.05))
    x = rnd((4, 2600), 2, torch.bfloat16)
    y = lin(x, y_f32=True)
    ref, mag = of.linear(f32(x), f32(lin.codes), f32(lin.scales))
    near(f64(y), ref, _tol_gemm(mag, 2600, torch.float32, ref))
    lin = Fp8Linear.from_weight(rnd((4864, 4864), 3, torch.bfloat16, 0.05))
    x, dy = rnd((130, 4864), 4, torch.bfloat16), rnd((130, 4864), 5, torch.bfloat16)
    dx, dw = lin.vjp(x, dy)
    _err_ok()
    rx, mx, rw, mw = of.vjp(f32(x), f32(dy), f32(lin.codes), f32(lin.scales))
    near(f64(dx), rx, _tol_gemm(mx, 4864, torch.bfloat16, rx), "dx")
    near(f64(dw), rw, _tol_gemm(mw, 130, torch.float32, rw), "dw")


def _tile(M, N, rows=0, accumulate=0):
    import ctypes
    from gsq_rco_mlx_b200 import _lib
    r, c = ctypes.c_int(), ctypes.c_int()
    _lib.check(_lib.load().gsq_fp8_gemm_tile(M, N, rows, accumulate, _lib.num_sms(), 1,
                                             ctypes.byref(r), ctypes.byref(c)), "tile")
    return r.value, c.value


def _product(a, b):
    """(a b^T, the sum of the products' magnitudes) of float64 arrays, in 64 bits."""
    a, b = torch.from_numpy(a).cuda(), torch.from_numpy(b).cuda()
    return (a @ b.t()).cpu().numpy(), (a.abs() @ b.abs().t()).cpu().numpy()


# sizes that the rule gives each tile of 128 rows or more, with more tiles than pairs (or CTAs),
# ten ragged blocks of 128 along the sum, and ragged last tiles
TILES = [(2047, 4864, 0, (256, 256)), (1300, 4000, 0, (256, 256)), (100, 19000, 0, (128, 128)),
         (1400, 3200, 0, (128, 128))]
TILES_ROWS = [(3000, 3000, 1, (256, 256)), (1300, 4000, 1, (128, 128)), (100, 19000, 1, (128, 128))]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("M,N,rows,tile", TILES)
def test_fp8_linear_in_every_tile(M, N, rows, tile, dtype):
    """Each k-block's own scales, the stages' and the scale ring's second turn, outputs of every
    type on 16 bytes (written in boxes) and off them (value by value)."""
    from gsq_rco_mlx_b200.common.fp8 import Fp8Linear, quantize_rows
    K = 1200
    assert _tile(M, N, rows) == tile and -(-M // tile[0]) * -(-N // tile[1]) > \
        (148 if tile[0] == 128 else 74)
    lin = Fp8Linear.from_weight(rnd((N, K), 1, scale=0.05) * torch.exp(rnd((N, K), 8)[:, :1]))
    x = rnd((M, K), 2, DT[dtype])
    y, y32, yq = lin(x), lin(x, y_f32=True), lin(quantize_rows(x))
    buf = torch.full((M, N + 5), 7.0, device="cuda", dtype=DT[dtype])
    lin(x, out=buf[:, 3:3 + N])
    _err_ok()
    assert torch.equal(buf[:, 3:3 + N], y)
    assert bool((buf[:, :3] == 7).all()) and bool((buf[:, 3 + N:] == 7).all())
    ref, mag = _product(of.rows_value(*of.quantize_rows(f32(x))),
                        of.blocks_value(f32(lin.codes), f32(lin.scales)))
    for got in (y, y32, yq):
        near(f64(got), ref, _tol_gemm(mag, K, got.dtype, ref))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("N,K,rows,tile", TILES_ROWS)
def test_fp8_weight_gradient_in_every_tile(N, K, rows, tile, dtype):
    """The same of dW (a scale per row of both sides), written and added to what is there, on 16
    bytes and off them; and of dx from it."""
    from gsq_rco_mlx_b200.common.fp8 import Fp8Linear
    M = 1200
    assert _tile(N, K, rows) == _tile(N, K, rows, accumulate=1) == tile
    lin = Fp8Linear.from_weight(rnd((N, K), 3, scale=0.05), transposed=True)
    x = rnd((M, K), 4, DT[dtype]) * torch.exp(rnd((M, 1), 6)).to(DT[dtype])
    dy = rnd((M, N), 5, DT[dtype], 0.01)
    dx, dw = lin.vjp(x, dy)
    base = rnd((N, K), 7)
    acc = base.clone()
    lin.vjp(x, dy, dw=acc, accumulate=True)
    buf = torch.full((N, K + 7), 7.0, device="cuda")
    buf[:, 5:5 + K] = base
    lin.vjp(x, dy, dw=buf[:, 5:5 + K], accumulate=True)
    _err_ok()
    assert torch.equal(buf[:, 5:5 + K], acc)
    assert bool((buf[:, :5] == 7).all()) and bool((buf[:, 5 + K:] == 7).all())
    lin.vjp(x, dy, dw=buf[:, 5:5 + K])
    assert torch.equal(buf[:, 5:5 + K], dw)
    wv = of.blocks_value(f32(lin.codes), f32(lin.scales))
    rx, mx = _product(of.rows_value(*of.quantize_rows(f32(dy))), np.ascontiguousarray(wv.T))
    near(f64(dx), rx, _tol_gemm(mx, N, DT[dtype], rx), "dx")
    rw, mw = _product(of.rows_value(*of.quantize_rows(np.ascontiguousarray(f32(dy).T))),
                      of.rows_value(*of.quantize_rows(np.ascontiguousarray(f32(x).T))))
    near(f64(dw), rw, _tol_gemm(mw, M, torch.float32, rw), "dw")
    total = rw + f64(base)
    near(f64(acc), total, _tol_gemm(mw, M, torch.float32, rw) + U * np.abs(total), "dw added")


@pytest.mark.parametrize("M", [13, 30, 64])
def test_fp8_few_rows_long_sums(M):
    """Each few-row kernel with more k-blocks a CTA than it has stages (5), accumulators (4) and
    scales staged at a time (16): 21, not shared out; and 41 over a cluster."""
    from gsq_rco_mlx_b200.common.fp8 import Fp8Linear
    for K, N in ((2600, 19000), (5200, 3000)):
        assert _tile(M, N) == (16 if M <= 16 else 32 if M <= 32 else 64, 128)
        lin = Fp8Linear.from_weight(rnd((N, K), 1, torch.bfloat16, 0.05))
        x = rnd((M, K), 2, torch.bfloat16) * torch.exp(rnd((M, K), 3)[:, :1]).bfloat16()
        y = lin(x, y_f32=True)
        _err_ok()
        ref, mag = of.linear(f32(x), f32(lin.codes), f32(lin.scales))
        near(f64(y), ref, _tol_gemm(mag, K, torch.float32, ref))


def test_fp8_strides_outputs_and_refusals():
    """Rows of a wider buffer, a transposed input, outputs inside a wider buffer (whose other
    columns stay), no rows at all; and what is refused."""
    from gsq_rco_mlx_b200.common.fp8 import Fp8Linear, Fp8Tensor, quantize_rows
    K, N = 200, 130
    lin = Fp8Linear.from_weight(rnd((N, K), 7))
    wide = rnd((9, 333), 8, torch.bfloat16)
    x = wide[:, 7:7 + K]
    buf = torch.full((9, 200), 7.0, device="cuda", dtype=torch.bfloat16)
    lin(x, out=buf[:, 3:3 + N])
    want = lin(x.contiguous())
    assert torch.equal(buf[:, 3:3 + N], want)
    assert bool((buf[:, :3] == 7).all()) and bool((buf[:, 3 + N:] == 7).all())
    xt = x.t().contiguous().t()
    assert torch.equal(lin(xt), want)
    # rows of a quantized tensor (scales of a larger pitch), one of them, and from its first block
    q = quantize_rows(x)
    for r0, r1 in ((2, 7), (4, 5), (0, 9)):
        part = Fp8Tensor(q.codes[r0:r1], q.scales[r0:r1])
        assert torch.equal(lin(part), want[r0:r1]), (r0, r1)
    e = lin(x[:0])
    assert e.shape == (0, N)
    dx, dw = lin.vjp(x[:0], want[:0])
    assert dx.shape == (0, K) and not bool(dw.any())
    W = torch.empty(N, K, device="cuda", dtype=torch.bfloat16)
    lin.dequant(W)
    # a weight whose rows are not on 16 bytes, and scales of other strides
    c = torch.zeros(N, K + 3, device="cuda", dtype=torch.uint8)
    c[:, 3:] = lin.codes.view(torch.uint8)
    other = Fp8Linear(c[:, 3:].view(torch.float8_e4m3fn), lin.scales.t().contiguous().t())
    assert torch.equal(other(x), want)
    for bad in (lambda: lin(x[:, :K - 1]), lambda: lin(x.double()), lambda: lin(x.cpu()),
                lambda: lin(x, out=buf), lambda: lin(x, out=buf[:, :N].float()),
                lambda: lin(x.reshape(1, 9, K)), lambda: lin.vjp(x, want[:8]),
                lambda: lin.vjp(x, want, accumulate=True),
                lambda: lin.vjp(x, want, dw=torch.empty(N, K, device="cuda").half()),
                lambda: lin(quantize_rows(x[:, :K - 1])),
                lambda: Fp8Linear(lin.codes, lin.scales[:1]),
                lambda: Fp8Linear(lin.codes, lin.scales.double()),
                lambda: Fp8Linear(lin.codes.view(torch.uint8), lin.scales),
                lambda: Fp8Linear(lin.codes, lin.scales, codes_t=lin.codes),
                lambda: Fp8Tensor(lin.codes, lin.scales)):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("M", [3, 200])
def test_fp8_not_finite_and_extreme_values(M):
    """NaN or infinity in a row reaches that row only; zeros, denormals and the type's largest
    values stay finite where the product does."""
    from gsq_rco_mlx_b200.common.fp8 import Fp8Linear
    K, N = 300, 140
    lin = Fp8Linear.from_weight(rnd((N, K), 9))
    x = rnd((M, K), 10)
    clean = lin(x)
    x2 = x.clone()
    x2[1, 290] = float("inf")
    x2[2, 5] = float("nan")
    y = lin(x2)
    _err_ok()
    assert bool(torch.isnan(y[1:3]).all())
    assert torch.equal(y[0], clean[0]) and torch.equal(y[3:], clean[3:])
    z = torch.zeros(M, K, device="cuda")
    assert not bool(lin(z).any())
    z[:, ::2] = 1e-42   # denormal: below the floor of the scale, rounds to zero codes
    assert not bool(lin(z).any())
    big = torch.full((M, K), 3e37, device="cuda")
    ref, mag = of.linear(f32(big), f32(lin.codes), f32(lin.scales))
    # 300 products of 3e37 and weights of order 1 add up to 5e38 and more, beyond float32's
    # 3.4e38, where infinity is the right answer. Whatever the order in which the three blocks'
    # sums c_b are added: every partial sum is at most sum |c_b|, so the output is finite where
    # that fits; and no order makes a finite number of an exact sum that does not fit. (The sum
    # inside a block is in units of the codes, at most 128 * 448^2.)
    xv = of.rows_value(*of.quantize_rows(f32(big)))
    wv = of.blocks_value(f32(lin.codes), f32(lin.scales))
    most = float(np.finfo(np.float32).max)
    part = sum(np.abs(xv[:, a:a + 128] @ wv[:, a:a + 128].T) for a in range(0, K, 128)) / most
    got = f64(lin(big))
    fits, over = part < 1 - 1e-4, np.abs(ref) / most > 1 + 1e-4
    assert fits.any() and over.any() and not np.isfinite(got[over]).any()
    near(got[fits], ref[fits], _tol_gemm(mag, K, torch.float32, ref)[fits])


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("M", [5, 200])
def test_fp8_gradients_of_values_that_are_not_finite(M, dtype):
    """A row of dy with NaN or infinity reaches its row of dx and its column's row of dW; one of x
    a column of dW. A block's values are NaN with it, so a token's whole block of 128 is."""
    from gsq_rco_mlx_b200.common.fp8 import Fp8Linear
    K, N = 300, 140
    lin = Fp8Linear.from_weight(rnd((N, K), 9, scale=0.05), transposed=True)
    x, dy = rnd((M, K), 4, DT[dtype]), rnd((M, N), 5, DT[dtype], 0.01)
    x[2, 290], dy[1, 7], dy[M - 1, 139] = float("inf"), float("nan"), float("-inf")
    dx, dw = lin.vjp(x, dy)
    _err_ok()
    nan_x, nan_w = np.zeros((M, K), bool), np.zeros((N, K), bool)
    nan_x[[1, M - 1]], nan_w[[7, 139]], nan_w[:, 290] = True, True, True
    assert np.array_equal(np.isnan(f64(dx)), nan_x) and np.array_equal(np.isnan(f64(dw)), nan_w)
    clean_x, clean_dy = x.clone(), dy.clone()
    clean_x[2, 290], clean_dy[1, 7], clean_dy[M - 1, 139] = 0, 0, 0
    rx, mx, rw, mw = of.vjp(f32(clean_x), f32(clean_dy), f32(lin.codes), f32(lin.scales))
    near(f64(dx)[~nan_x], rx[~nan_x], _tol_gemm(mx, N, DT[dtype], rx)[~nan_x], "dx")
    near(f64(dw)[~nan_w], rw[~nan_w], _tol_gemm(mw, M, torch.float32, rw)[~nan_w], "dw")


# ------------------------------------------------------------------------------------- rotary ---
SCALINGS = [None, {"type": "linear", "factor": 4.0}, {"type": "ntk", "factor": 8.0},
            {"type": "yarn", "factor": 8.0, "original": 4096},
            {"type": "bands", "factor": 8.0, "original": 8192}]


def _rope_tol(x, positions, w, rot, layout, factor, dtype, ref):
    """The remainder of the angle (in half turns) is rounded to float32 (2^-25 half turns, 2^-25 pi
    radians), the whole angle in 64 bits carries 4 2^-53 of itself; sine and cosine are good to 2
    steps (4 u), the factor and the two products and their sum round by u each."""
    a = np.abs(x)
    mag = a.copy()
    t = np.abs(np.asarray(positions, np.float64))[:, None]
    ang = np.zeros_like(a)
    for j in range(rot // 2):
        p, q = (j, j + rot // 2) if layout == "half" else (2 * j, 2 * j + 1)
        mag[..., p] = mag[..., q] = a[..., p] + a[..., q]
        ang[..., p] = ang[..., q] = 4 * 2.0 ** -53 * t * w[j]
    return factor * mag * (np.pi * 2.0 ** -25 + 8 * U + ang) + half(dtype) * np.abs(ref) + tiny(dtype)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("T,nq,nk,hd,rot", [(1, 14, 2, 64, 64), (1, 1, 0, 2, 2), (7, 8, 1, 128, 64),
                                            (33, 3, 3, 80, 20), (513, 4, 2, 96, 96),
                                            (5, 2, 1, 33, 6), (2, 7, 1, 256, 128),
                                            (70, 64, 8, 128, 128)])
def test_rotary(T, nq, nk, hd, rot, layout, dtype):
    from gsq_rco_mlx_b200.common.rotary import Rotary
    d = DT[dtype]
    sc = SCALINGS[(T + nq + hd) % len(SCALINGS)]
    r = Rotary(hd, 1e6, rot, layout, sc)
    packed = rnd((T, (nq + 2 * nk) * hd), T, d)
    q = packed[:, :nq * hd].view(T, nq, hd)
    k = packed[:, nq * hd:(nq + nk) * hd].view(T, nk, hd) if nk else None
    rng = np.random.default_rng(T)
    pos = rng.integers(-5, 4000000, T)
    pos[0] = 2 ** 31 - 1 if T > 1 else 1000003
    p = torch.from_numpy(pos).cuda()
    keep = packed.clone()
    for inverse in (False, True):
        f = r.vjp if inverse else r
        qo, ko = f(q, k, p.int() if pos.max() < 2 ** 31 else p)
        for x, o in ((q, qo), (k, ko)):
            if x is None:
                assert o is None
                continue
            ref = ob.rotate(f64(x), pos, r.freqs, rot, layout, r.factor, inverse)
            near(f64(o), ref, _rope_tol(f64(x), pos, r.freqs, rot, layout, r.factor, d, ref))
            assert torch.equal(o[..., rot:], x[..., rot:])
        q64, _ = f(q, k, p)   # int64 positions: the same bits
        assert torch.equal(q64, qo)
    assert torch.equal(packed, keep)
    # in place on the packed rows: q and k as above, v untouched
    qo, ko = r(q, k, p)
    r(q, k, p, out=(q, k))
    assert torch.equal(q, qo) and (k is None or torch.equal(k, ko))
    assert torch.equal(packed[:, (nq + nk) * hd:], keep[:, (nq + nk) * hd:])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("T,nq,nk,hd,rot", [(1024, 14, 2, 64, 64), (4096, 14, 2, 64, 64),
                                            (300, 32, 8, 128, 64), (2500, 7, 1, 80, 20)])
def test_rotary_gives_a_token_the_same_bits_in_any_batch(T, nq, nk, hd, rot, layout):
    """However many heads a thread turns, which goes by the number of tokens and heads."""
    from gsq_rco_mlx_b200.common.rotary import Rotary
    r = Rotary(hd, 1e6, rot, layout, SCALINGS[4])
    q, k = rnd((T, nq, hd), 1, torch.bfloat16), rnd((T, nk, hd), 2, torch.bfloat16)
    p = torch.arange(T, device="cuda") * 37
    qo, ko = r(q, k, p)
    for t in (0, T // 2, T - 1):
        for n in (1, 64):
            a, b = r(q[t:t + n], k[t:t + n], p[t:t + n])
            assert torch.equal(a, qo[t:t + n]) and torch.equal(b, ko[t:t + n])
    for h in (0, nq - 1):
        assert torch.equal(r(q[:, h:h + 1], None, p)[0], qo[:, h:h + 1])


def test_rotary_far_positions_and_layouts():
    """int64 positions beyond 2^31, head-major buffers, unaligned rows, a broadcast key input."""
    from gsq_rco_mlx_b200.common.rotary import Rotary
    r = Rotary(64, 1e6)
    T = 19
    pos = np.arange(T) + 5 * 2 ** 32
    p = torch.from_numpy(pos).cuda()
    hm = rnd((3, T, 64), 1).transpose(0, 1)
    q, _ = r(hm, None, p)
    ref = ob.rotate(f64(hm), pos, r.freqs, 64, "half")
    near(f64(q), ref, _rope_tol(f64(hm), pos, r.freqs, 64, "half", 1.0, torch.float32, ref))
    odd = rnd((T, 3 * 65 + 1), 2, torch.float16)
    v = odd[:, 1:].view(T, 3, 65)[:, :, :64] if odd[:, 1:].is_contiguous() else \
        torch.as_strided(odd, (T, 3, 64), (3 * 65 + 1, 65, 1), 1)
    assert torch.equal(r(v, None, p)[0], r(v.contiguous(), None, p)[0])
    k1 = rnd((T, 1, 64), 3).expand(T, 4, 64)   # a shared key head read four times
    _, ko = r(hm, k1, p)
    assert torch.equal(ko, r(hm, k1.contiguous(), p)[1])
    out = torch.zeros(3, T, 64, device="cuda").transpose(0, 1)
    r(hm, None, p, out=(out, None))
    assert torch.equal(out, q)
    e, _ = r(hm[:0], None, p[:0])
    assert e.shape == (0, 3, 64)
    for bad in (lambda: r(hm, None, p[:-1]), lambda: r(hm, None, p.float()),
                lambda: r(hm, None, p.cpu()), lambda: r(hm, hm.half(), p),
                lambda: r(hm[..., :32], None, p), lambda: r(hm, hm[:5], p),
                lambda: r(hm, hm, p, out=(out, None)),
                lambda: r(hm, None, p, out=(k1, None)),
                lambda: r(hm[:, :0], None, p),
                lambda: r(torch.zeros(T, 64, 3, device="cuda").transpose(1, 2), None, p),
                lambda: r(hm, None, p, out=(torch.as_strided(hm, (T, 3, 64), (192, 64, 1)), None))):
        with pytest.raises(ValueError):
            bad()


def test_rotary_refuses_outputs_across_its_inputs():
    """Outputs over other rows than their own input's; in place and beside, as usual buffers lie."""
    from gsq_rco_mlx_b200.common.rotary import Rotary
    r, T = Rotary(64, 1e6), 6
    p = torch.arange(T, device="cuda") + 9
    buf = rnd((T + 2, 8 * 64), 3, torch.bfloat16)
    part = lambda b, t, h, n: b.view(T + 2, 8, 64)[t:t + T, h:h + n]  # noqa: E731
    q, k = part(buf, 0, 0, 2), part(buf, 0, 2, 2)
    want = r(q, k, p)
    keep = buf.clone()
    for f in (r, r.vjp):
        for out in ((k, q), (part(buf, 1, 0, 2), want[1]), (want[0], part(buf, 0, 1, 2)),
                    (want[0], want[0]), (q, part(buf, 0, 1, 2))):
            with pytest.raises(ValueError, match="overlaps"):
                f(q, k, p, out=out)
    assert torch.equal(buf, keep)
    for h, g in ((0, 2), (4, 6), (4, 2)):   # in place, behind them in the same rows, one of both
        b = buf.clone()
        qb, kb = part(b, 0, 0, 2), part(b, 0, 2, 2)
        out = part(b, 0, h, 2), part(b, 0, g, 2)
        r(qb, kb, p, out=out)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    heads = buf[:, :2 * 64].reshape(T + 2, 2, 64).transpose(0, 1).contiguous().transpose(0, 1)[:T]
    assert torch.equal(r(heads, None, p, out=(heads, None))[0], want[0])


def test_rotary_values_that_are_not_finite():
    """NaN and infinity stay inside their pair."""
    from gsq_rco_mlx_b200.common.rotary import Rotary
    r = Rotary(16, 1e4, 8, "interleaved")
    q = rnd((3, 2, 16), 4)
    p = torch.arange(3, device="cuda")
    clean, _ = r(q, None, p)
    q[1, 0, 3] = float("nan")
    q[2, 1, 15] = float("inf")
    o, _ = r(q, None, p)
    assert bool(torch.isnan(o[1, 0, 2:4]).all()) and float(o[2, 1, 15]) == float("inf")
    same = torch.ones_like(o, dtype=torch.bool)
    same[1, 0, 2:4] = False
    same[2, 1, 15] = False
    assert torch.equal(o[same], clean[same])


# ------------------------------------------------------------------------------ residual norms ---
def _norm_inputs(T, H, dtype, post, pre, gates, seed=0):
    d = DT[dtype]
    v = {"h": rnd((T, H), seed + 1, d, 2.0), "y": rnd((T, H), seed + 2, d)}
    v["w_post"] = (1 + rnd((H,), seed + 3, scale=0.2)).to(d) if post else None
    v["w_pre"] = (1 + rnd((H,), seed + 4, scale=0.2)).to(d) if pre else None
    v["gate"] = rnd((gates, H), seed + 5, d) if gates else None
    v["dh"] = rnd((T, H), seed + 6, d)
    v["dx"] = rnd((T, H), seed + 7, d) if pre else None
    return v


def _o(v):
    return {k: None if t is None else f64(t) for k, t in v.items()}


NORMS = [(1, 1, True, True, 0), (1, 896, True, True, 1), (5, 128, False, True, 0),
         (6, 257, True, False, 3), (33, 896, True, True, 0), (40, 1000, True, True, 40),
         (12, 1025, False, True, 4), (9, 2048, True, True, 1), (7, 4097, True, True, 7),
         (1200, 64, True, True, 2), (3, 8192, True, False, 1), (2, 12345, True, True, 1),
         (2, 32768, True, True, 2), (2500, 100, False, True, 1), (3, 5, True, True, 3)]


def _check_norm(v, h2, x, stats, scale, eps, off):
    """The squares' sum adds at most 32 values a thread, 32 threads and 32 warps in trees or
    chains of at most 48 roundings; half of it reaches the reciprocal root, which rounds by 4 u
    more; then at most 6 products: 40 u covers n, and once more x. Returns the exact x and the
    bound on it before its own rounding."""
    o, d = _o(v), v["h"].dtype
    rh, rx, r1, r2, n = ob.residual_norm(o["h"], o["y"], o["w_post"], o["w_pre"], o["gate"], scale,
                                         eps, off)
    hm = np.abs(o["h"]) + np.abs(rh - o["h"])
    near(f64(h2), rh, 40 * U * hm + half(d) * np.abs(rh) + tiny(d), "h")
    # r2 moves by the relative error of the root mean square of h'
    e2 = 40 * U * (1 + np.sqrt((hm ** 2).mean(1, keepdims=True)) * r2)
    near(f64(stats), np.stack([r1[:, 0], r2[:, 0]]),
         np.stack([40 * U * r1[:, 0], (e2 * r2)[:, 0] if rx is not None else 0 * r2[:, 0]]), "stats")
    if rx is None:
        assert x is None
        return None, None
    xt = 40 * U * hm * r2 * np.abs(o["w_pre"] + off) + e2 * np.abs(rx)
    near(f64(x), rx, xt + half(d) * np.abs(rx) + tiny(d), "x")
    return rx, xt


def _check_norm_vjp(v, g, dh, scale, eps, off):
    """Along a row: the statistics carry 40 u, each mean of products at most 48 roundings more and
    there are two of them, each formed from at most 12 products: 200 u of the magnitudes (of the
    first gradient, and once more through the second). Over rows: one rounding a row at most."""
    o, d = _o(v), v["h"].dtype
    ref, mag = ob.residual_norm_vjp(o["h"], o["y"], o["w_post"], o["w_pre"],
                                    None if dh is None else o["dh"], o["dx"], o["gate"], scale,
                                    eps, off)
    for name in ("dh", "dy", "dw_post", "dw_pre", "dgate"):
        if name not in ref:
            assert g[name] is None
        elif name in ("dh", "dy"):
            near(f64(g[name]), ref[name],
                 400 * U * mag[name] + half(d) * np.abs(ref[name]) + tiny(d), name)
        else:
            assert g[name].dtype == torch.float32
            near(f64(g[name]), ref[name], (400 + v["h"].shape[0]) * U * mag[name], name)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("T,H,post,pre,gates", NORMS)
def test_residual_norm(T, H, post, pre, gates, dtype):
    from gsq_rco_mlx_b200.common.norm import residual_norm
    d = DT[dtype]
    v = _norm_inputs(T, H, dtype, post, pre, gates)
    off = 0.0 if T % 2 else 1.0
    h2, x, stats = residual_norm(v["h"], v["y"], v["w_post"], v["w_pre"], gate=v["gate"], scale=0.7,
                                 eps=1e-5, offset=off)
    rx, xt = _check_norm(v, h2, x, stats, 0.7, 1e-5, off)
    if not pre:
        return
    h3, q, s3 = residual_norm(v["h"], v["y"], v["w_post"], v["w_pre"], gate=v["gate"], scale=0.7,
                              eps=1e-5, offset=off, fp8=True)
    assert torch.equal(h3, h2) and torch.equal(s3, stats)
    # the codes' values within half a step of x (2^-4, or 2^-10 of the scale), x as above
    sc = np.repeat(f64(q.scales), 128, 1)[:, :H]
    near(f64(q.float()), rx, xt + np.maximum(2.0 ** -4 * (np.abs(rx) + xt), 2.0 ** -10 * sc)
         * (1 + 2.0 ** -18) + 2.0 ** -22 * np.abs(rx), "e4m3")
    amax = np.abs(np.pad(rx, ((0, 0), (0, -H % 128)))).reshape(T, -1, 128).max(2)
    xm = np.pad(xt, ((0, 0), (0, -H % 128))).reshape(T, -1, 128).max(2)
    near(f64(q.scales), np.maximum(amax, 2.0 ** -100) / 448, (xm + 2 * U * amax) / 448, "scales")


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("T,H,post,pre,gates", NORMS)
def test_residual_norm_vjp(T, H, post, pre, gates, dtype):
    from gsq_rco_mlx_b200.common.norm import residual_norm, residual_norm_vjp
    d = DT[dtype]
    v = _norm_inputs(T, H, dtype, post, pre, gates, seed=20)
    off = 1.0 if T % 2 else 0.0
    _, _, stats = residual_norm(v["h"], v["y"], v["w_post"], v["w_pre"], gate=v["gate"], scale=0.7,
                                eps=1e-5, offset=off)
    dh = None if (T % 3 == 0 and pre) else v["dh"]
    g, again = (residual_norm_vjp(v["h"], v["y"], v["w_post"], v["w_pre"], stats, dh, v["dx"],
                                  gate=v["gate"], scale=0.7, offset=off) for _ in range(2))
    _check_norm_vjp(v, g, dh, 0.7, 1e-5, off)
    assert all(g[n] is None or torch.equal(g[n], again[n]) for n in g)
    _err_ok()


# more rows than teams, so that a team's ring of rows turns more than once and its next row is read
# ahead; more gate rows than teams; each way of holding the weights, on 16 bytes and off them
MANY = [(20000, 200, 1), (20000, 100, 0), (6000, 128, 6000), (6000, 896, 3000), (6000, 900, 2),
        (1500, 2048, 1), (1200, 5121, 3), (1500, 6400, 500), (1300, 7001, 0), (700, 9000, 350)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("T,H,gates", MANY)
def test_residual_norm_many_rows_a_team(T, H, gates, dtype):
    from gsq_rco_mlx_b200.common.norm import residual_norm, residual_norm_vjp
    v = _norm_inputs(T, H, dtype, True, True, gates, seed=60)
    args, kw = (v["w_post"], v["w_pre"]), dict(gate=v["gate"], scale=0.7)
    h2, x, st = residual_norm(v["h"], v["y"], *args, eps=1e-5, **kw)
    rx, xt = _check_norm(v, h2, x, st, 0.7, 1e-5, 0.0)
    h3, q, s3 = residual_norm(v["h"], v["y"], *args, eps=1e-5, fp8=True, **kw)
    assert torch.equal(h3, h2) and torch.equal(s3, st)
    sc = np.repeat(f64(q.scales), 128, 1)[:, :H]
    near(f64(q.float()), rx, xt + np.maximum(2.0 ** -4 * (np.abs(rx) + xt), 2.0 ** -10 * sc)
         * (1 + 2.0 ** -18) + 2.0 ** -22 * np.abs(rx), "e4m3")
    over = v["h"].clone()   # in place, the next row read ahead
    assert torch.equal(residual_norm(over, v["y"], *args, eps=1e-5, out=over, **kw)[1], x)
    assert torch.equal(over, h2)
    g, again = (residual_norm_vjp(v["h"], v["y"], *args, st, v["dh"], v["dx"], **kw)
                for _ in range(2))
    _check_norm_vjp(v, g, v["dh"], 0.7, 1e-5, 0.0)
    assert all(g[n] is None or torch.equal(g[n], again[n]) for n in g)
    _err_ok()


def test_residual_norm_rows_strides_and_refusals():
    """Rows of wider and odd buffers, h updated in place, rows behind the last left alone, a row of
    zeros, values that are not finite, no rows; and what is refused."""
    from gsq_rco_mlx_b200.common.norm import residual_norm, residual_norm_vjp
    T, H = 6, 200
    v = _norm_inputs(T, H, "bf16", True, True, 2)
    kw = dict(gate=v["gate"], scale=0.5)
    args = (v["w_post"], v["w_pre"])
    h2, x, st = residual_norm(v["h"], v["y"], *args, **kw)
    for pad in (8, 3):
        wide = torch.full((T + 2, H + pad), 9.0, device="cuda", dtype=torch.bfloat16)
        rows = wide[:T, pad:]
        rows.copy_(v["h"])
        out, x2, st2 = residual_norm(rows, v["y"], *args, out=rows, **kw)
        assert out.data_ptr() == rows.data_ptr()
        if pad == 8:   # rows on 16 bytes: the same sums in the same order
            assert torch.equal(rows, h2) and torch.equal(x2, x) and torch.equal(st2, st)
        _check_norm(v, rows, x2, st2, 0.5, 1e-6, 0.0)
        assert bool((wide[T:] == 9).all()) and bool((wide[:, :pad] == 9).all())
        rows.copy_(v["h"])
        g = residual_norm_vjp(rows, v["y"], *args, st, v["dh"], v["dx"], **kw)
        if pad == 8:
            want = residual_norm_vjp(v["h"], v["y"], *args, st, v["dh"], v["dx"], **kw)
            assert all(torch.equal(g[n], want[n]) for n in g)
        _check_norm_vjp(v, g, v["dh"], 0.5, 1e-6, 0.0)
    z = torch.zeros_like(v["h"])
    h0, x0, s0 = residual_norm(z, z, *args, **kw)
    assert not bool(h0.any()) and not bool(x0.any())
    near(f64(s0), np.full((2, T), 1e3), 4 * U * 1e3)
    bad = v["y"].clone()
    bad[1, 7], bad[3, 0] = float("nan"), float("inf")
    h3, x3, _ = residual_norm(v["h"], bad, *args, **kw)
    ok = [0, 2, 4, 5]
    assert torch.equal(h3[ok], h2[ok]) and torch.equal(x3[ok], x[ok])
    assert bool(torch.isnan(x3[[1, 3]]).any(1).all())
    one, xo, _ = residual_norm(v["h"], v["y"], *args, gate=v["gate"][0], scale=0.5)
    assert torch.equal(one[:3], h2[:3]) and torch.equal(xo[:3], x[:3])
    e = residual_norm(v["h"][:0], v["y"][:0], *args, gate=v["gate"][0])
    assert e[0].shape == (0, H) and e[2].shape == (2, 0)
    ge = residual_norm_vjp(v["h"][:0], v["y"][:0], *args, e[2], v["dh"][:0], v["dx"][:0],
                           gate=v["gate"][0])
    assert not bool(ge["dw_pre"].any()) and ge["dgate"].shape == (H,)
    f = residual_norm
    for call in (lambda: f(v["h"], v["y"][:5], *args), lambda: f(v["h"], v["y"].float(), *args),
                 lambda: f(v["h"], v["y"], v["w_post"][:9]), lambda: f(v["h"].double(), v["y"]),
                 lambda: f(v["h"], v["y"], *args, gate=v["gate"].float()),
                 lambda: f(v["h"], v["y"], *args, gate=torch.zeros(4, H, device="cuda").bfloat16()),
                 lambda: f(v["h"], v["y"], v["w_post"], fp8=True), lambda: f(v["h"].cpu(), v["y"]),
                 lambda: f(v["h"], v["y"], v["w_post"].cpu()),
                 lambda: f(v["h"], v["y"], *args, out=h2.float()),
                 lambda: f(torch.zeros(1, 32769, device="cuda"), torch.zeros(1, 32769, device="cuda"),
                           torch.zeros(32769, device="cuda")),
                 lambda: residual_norm_vjp(v["h"], v["y"], *args, st[:, :5], v["dh"], v["dx"]),
                 lambda: residual_norm_vjp(v["h"], v["y"], *args, st, v["dh"], None),
                 lambda: residual_norm_vjp(v["h"], v["y"], v["w_post"], None, st, v["dh"], v["dx"]),
                 lambda: residual_norm_vjp(v["h"], v["y"], v["w_post"], None, st, None, None)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("T,H", [(6, 200), (6, 257), (5, 1000), (4, 1025), (7, 5124), (6, 9001)])
def test_residual_norm_values_that_are_not_finite(T, H, dtype):
    """NaN and infinity in h, y and the cotangents, in each kernel's rows: the values of the formula
    in 64 bits (infinity times a reciprocal root of zero is NaN), also in e4m3, where a block with
    one NaN is NaN; other rows as without them; the sums over rows NaN where a row is."""
    from gsq_rco_mlx_b200.common.norm import residual_norm, residual_norm_vjp
    v = _norm_inputs(T, H, dtype, True, True, 1, seed=40)
    args = (v["w_post"], v["w_pre"])
    kw = dict(gate=v["gate"], scale=0.5)
    clean = residual_norm(v["h"], v["y"], *args, **kw)
    c8 = residual_norm(v["h"], v["y"], *args, fp8=True, **kw)[1]
    _, _, st = clean
    g0 = residual_norm_vjp(v["h"], v["y"], *args, st, v["dh"], v["dx"], **kw)
    h, y = v["h"].clone(), v["y"].clone()
    h[0, 3], h[1, H - 1], y[2, 150], y[3, 0] = (float(n) for n in ("nan", "inf", "nan", "-inf"))
    h2, x, st2 = residual_norm(h, y, *args, **kw)
    q = residual_norm(h, y, *args, fp8=True, **kw)[1]
    # rows 0, 2: r1 or h' is NaN, so all of x is; row 1: h' holds one infinity, r2 is 0 and x is 0 but
    # for inf 0 = NaN; row 3: r1 is 0, the norm of y is 0 but for NaN at its infinity
    wide = np.ones((T, H), bool)
    one = np.zeros((T, H), bool)
    one[0, 3], one[2], one[3, 0] = True, True, True
    assert np.array_equal(np.isnan(f64(h2)), one)
    assert np.isinf(f64(h2)[1]).tolist() == [False] * (H - 1) + [True]
    nan = np.zeros((T, H), bool)
    nan[[0, 2, 3]], nan[1, H - 1] = True, True
    assert np.array_equal(np.isnan(f64(x)), nan) and not f64(x)[1, :H - 1].any()
    blocks = np.zeros((T, H), bool)
    blocks[[0, 2, 3]], blocks[1, (H - 1) // 128 * 128:] = True, True
    assert np.array_equal(np.isnan(f64(q.float())), blocks & wide)
    assert not f64(q.float())[1, :(H - 1) // 128 * 128].any()
    assert torch.equal(h2[4:], clean[0][4:]) and torch.equal(x[4:], clean[1][4:])
    assert torch.equal(q.codes[4:].view(torch.uint8), c8.codes[4:].view(torch.uint8))
    assert torch.equal(q.scales[4:], c8.scales[4:]) and torch.equal(st2[:, 4:], st[:, 4:])
    # the gradient: one NaN of a cotangent reaches its row, and every sum over rows where it is
    dh, dx = v["dh"].clone(), v["dx"].clone()
    dx[0, 5], dh[2, H - 2] = float("nan"), float("inf")
    g = residual_norm_vjp(v["h"], v["y"], *args, st, dh, dx, **kw)
    _err_ok()
    for n in ("dh", "dy"):
        assert torch.equal(g[n][3:], g0[n][3:]) and torch.equal(g[n][1], g0[n][1]), n
        assert bool(torch.isnan(g[n][0]).all())
    assert bool(torch.isinf(g["dh"][2, H - 2])) and bool(torch.isnan(g["dy"][2]).any())
    keep = torch.ones(H, dtype=torch.bool)
    keep[5] = False
    assert bool(torch.isnan(g["dw_pre"][5])) and torch.equal(g["dw_pre"][keep], g0["dw_pre"][keep])
    for n in ("dw_post", "dgate"):
        assert bool(torch.isnan(g[n]).all()), n


# ---------------------------------------------------------------------------- beyond 32 bits ---
@pytest.fixture
def give_back():
    """The tens of GB that a test took, to the device."""
    yield
    torch.cuda.empty_cache()


def test_norms_past_32_bit_offsets(give_back):
    """2.3e9 elements a tensor: the last rows as of a call on them alone (same width, same kernel)."""
    from gsq_rco_mlx_b200.common.norm import residual_norm, residual_norm_vjp
    T, H, n = 70000, 32768, 5
    g = torch.Generator(device="cuda").manual_seed(1)
    big = lambda: torch.empty(T, H, device="cuda", dtype=torch.bfloat16).normal_(generator=g)  # noqa: E731
    h, y = big(), big()
    w = rnd((H,), 3, torch.bfloat16)
    h2, q, st = residual_norm(h, y, w, w, fp8=True)
    a = residual_norm(h[-n:], y[-n:], w, w, fp8=True)
    assert torch.equal(h2[-n:], a[0]) and torch.equal(st[:, -n:], a[2])
    assert torch.equal(q.codes[-n:].view(torch.uint8), a[1].codes.view(torch.uint8))
    assert torch.equal(q.scales[-n:], a[1].scales)
    del h2, q
    grads = residual_norm_vjp(h, y, w, w, st, y, h)
    b = residual_norm_vjp(h[-n:], y[-n:], w, w, st[:, -n:], y[-n:], h[-n:])
    assert all(torch.equal(grads[k][-n:], b[k]) for k in ("dh", "dy"))
    _err_ok()


def test_rotary_past_32_bit_offsets(give_back):
    from gsq_rco_mlx_b200.common.rotary import Rotary
    T, n = 140000, 5
    g = torch.Generator(device="cuda").manual_seed(2)
    q = torch.empty(T, 128, 128, device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    r, pos = Rotary(128), torch.arange(T, device="cuda")
    want = r(q[-n:], None, pos[-n:])[0]
    heads = q[:T // 2].transpose(0, 1).contiguous().transpose(0, 1)   # head-major: 9e6 a head
    hw = r(q[T // 2 - n:T // 2], None, pos[T // 2 - n:T // 2])[0]
    r(heads, None, pos[:T // 2], out=(heads, None))
    r(q, None, pos, out=(q, None))
    assert torch.equal(q[-n:], want) and torch.equal(heads[-n:], hw)


def test_fp8_past_32_bit_offsets(give_back):
    """Rows of 2.5e9 elements through the product and its gradient, a weight of 2.2e9 both ways: some
    of the last rows and columns against the oracle. More rows and blocks than the quantization's
    and the dequantization's grids take in one go."""
    from gsq_rco_mlx_b200.common.fp8 import Fp8Linear
    g = torch.Generator(device="cuda").manual_seed(3)
    M, K, N, n = 300001, 8192, 130, 3
    x = torch.empty(M, K, device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    lin = Fp8Linear.from_weight(rnd((N, K), 4, scale=0.05), transposed=True)
    y = lin(x)
    ref, mag = of.linear(f32(x[-n:]), f32(lin.codes), f32(lin.scales))
    near(f64(y[-n:]), ref, _tol_gemm(mag, K, torch.bfloat16, ref), "y")
    dy = torch.empty(M, N, device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    dx, dw = lin.vjp(x, dy)
    _err_ok()
    wv = of.blocks_value(f32(lin.codes), f32(lin.scales))
    dv = of.rows_value(*of.quantize_rows(f32(dy[-n:])))
    near(f64(dx[-n:]), dv @ wv, _tol_gemm(np.abs(dv) @ np.abs(wv), N, torch.bfloat16, dv @ wv), "dx")
    a = of.rows_value(*of.quantize_rows(np.ascontiguousarray(f32(dy[:, -n:]).T)))
    b = of.rows_value(*of.quantize_rows(np.ascontiguousarray(f32(x[:, -n:]).T)))
    rw = a @ b.T
    near(f64(dw[-n:, -n:]), rw, _tol_gemm(np.abs(a) @ np.abs(b).T, M, torch.float32, rw), "dw")
    del x, y, dx
    N = 270001
    W = torch.empty(N, K, device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    lin = Fp8Linear.from_weight(W)
    q, s = of.quantize_blocks(f32(W[N // 128 * 128:]))   # the last block of rows
    m = N - N // 128 * 128
    assert np.array_equal(f32(lin.codes[-m:]), q) and np.array_equal(f32(lin.scales[-1:]), s)
    out = torch.empty_like(W)
    lin.dequant(out)
    v = of.blocks_value(q, s)
    near(f64(out[-m:]), v, (half(torch.bfloat16) + U) * np.abs(v) + tiny(torch.bfloat16))
    near(f64(out[:2]), of.blocks_value(*of.quantize_blocks(f32(W[:128])))[:2],
         (half(torch.bfloat16) + U) * np.abs(f64(out[:2])) * (1 + 2.0 ** -7) + tiny(torch.bfloat16))
    for rows in (1, 100):   # 2110 tiles of columns, the last one ragged
        z = rnd((rows, K), 6, torch.bfloat16)
        o = lin(z)
        ref, mag = of.linear(f32(z[-n:]), q, s)
        near(f64(o[-n:, -m:]), ref, _tol_gemm(mag, K, torch.bfloat16, ref), "wide")
    _err_ok()


# ------------------------------------------------------------------------------------ together ---
def _block(seed=0, H=256, T=300, heads=4, kv=2, hd=64):
    from gsq_rco_mlx_b200.common.fp8 import Fp8Linear
    from gsq_rco_mlx_b200.common.rotary import Rotary
    W = rnd(((heads + 2 * kv) * hd, H), seed, torch.bfloat16, 0.05)
    lin = Fp8Linear.from_weight(W, transposed=True)
    rot = Rotary(hd, 1e4, 32, "half", SCALINGS[3])
    v = _norm_inputs(T, H, "bf16", True, True, 1, seed)
    pos = torch.arange(T, device="cuda")
    return lin, rot, v, pos, heads, kv, hd


def _forward(lin, rot, v, pos, heads, kv, hd, fp8=True):
    from gsq_rco_mlx_b200.common.norm import residual_norm
    h2, x, st = residual_norm(v["h"], v["y"], v["w_post"], v["w_pre"], gate=v["gate"], scale=0.7,
                              fp8=fp8)
    qkv = lin(x)
    T = qkv.shape[0]
    q = qkv[:, :heads * hd].view(T, heads, hd)
    k = qkv[:, heads * hd:(heads + kv) * hd].view(T, kv, hd)
    qr, kr = rot(q, k, pos)
    return h2, x, st, qkv, qr, kr


def _backward(lin, rot, v, pos, heads, kv, hd, st, x, dq, dk, dv):
    """Cotangents of (q, k, v) back to h, y and every parameter."""
    from gsq_rco_mlx_b200.common.norm import residual_norm_vjp
    T = pos.shape[0]
    dqkv = torch.empty(T, (heads + 2 * kv) * hd, device="cuda", dtype=torch.bfloat16)
    rot.vjp(dq, dk, pos, out=(dqkv[:, :heads * hd].view(T, heads, hd),
                              dqkv[:, heads * hd:(heads + kv) * hd].view(T, kv, hd)))
    dqkv[:, (heads + kv) * hd:] = dv
    dx, dw = lin.vjp(x, dqkv)
    g = residual_norm_vjp(v["h"], v["y"], v["w_post"], v["w_pre"], st, v["dh"], dx,
                          gate=v["gate"], scale=0.7)
    return dict(g, dw=dw, dx=dx)


def test_norm_linear_rotary_in_a_row():
    """The norm into 8-bit rows, the projection and the rotation as a block runs them, each stage
    against the oracle on the stage's own inputs; the 8-bit rows are those of the float32 norm."""
    lin, rot, v, pos, heads, kv, hd = args = _block()
    h2, x, st, qkv, qr, kr = _forward(*args)
    _err_ok()
    wv = of.blocks_value(f32(lin.codes), f32(lin.scales))
    xv = f64(x.float())
    ref, mag = xv @ wv.T, np.abs(xv) @ np.abs(wv).T
    near(f64(qkv), ref, _tol_gemm(mag, 256, torch.bfloat16, ref), "qkv")
    for a, b, o in ((0, heads, qr), (heads, heads + kv, kr)):
        z = f64(qkv[:, a * hd:b * hd]).reshape(-1, b - a, hd)
        ref = ob.rotate(z, f64(pos), rot.freqs, 32, "half", rot.factor)
        near(f64(o), ref, _rope_tol(z, f64(pos), rot.freqs, 32, "half", rot.factor, torch.bfloat16,
                                    ref), "rotary")
    _, xb, _, qkvb, _, _ = _forward(*args, fp8=False)
    g = _backward(*args, st, xb, v["dh"].view(300, 4, 64), v["dx"][:, :128].reshape(300, 2, 64),
                  v["dx"][:, 128:])
    assert all(bool(torch.isfinite(t).all()) for t in g.values())


def test_a_training_step_backward_in_a_row():
    """norm -> projection -> rotation and back, as a training step calls them: the dense rows that
    the forward pass kept, the cotangents of q and k turned back where dqkv holds them. Each stage
    of the backward pass against the oracle on the stage's own inputs."""
    from gsq_rco_mlx_b200.common.norm import residual_norm, residual_norm_vjp
    lin, rot, v, pos, heads, kv, hd = args = _block(70)
    T, nq, nk = 300, heads * hd, kv * hd
    h2, x, st = residual_norm(v["h"], v["y"], v["w_post"], v["w_pre"], gate=v["gate"], scale=0.7)
    qkv = lin(x)
    q, k = qkv[:, :nq].view(T, heads, hd), qkv[:, nq:nq + nk].view(T, kv, hd)
    assert qkv.shape[1] == nq + 2 * nk
    rot(q, k, pos, out=(q, k))
    dqkv = rnd((T, nq + 2 * nk), 90, torch.bfloat16)
    got = dqkv.clone()   # cotangents of the turned q and k, and of v
    dq, dk = got[:, :nq].view(T, heads, hd), got[:, nq:nq + nk].view(T, kv, hd)
    rot.vjp(dq, dk, pos, out=(dq, dk))
    for a, n in ((0, heads), (nq, kv)):
        z = f64(dqkv[:, a:a + n * hd]).reshape(T, n, hd)
        ref = ob.rotate(z, f64(pos), rot.freqs, 32, "half", rot.factor, inverse=True)
        near(f64(got[:, a:a + n * hd]).reshape(T, n, hd), ref,
             _rope_tol(z, f64(pos), rot.freqs, 32, "half", rot.factor, torch.bfloat16, ref), "turned")
    assert torch.equal(got[:, nq + nk:], dqkv[:, nq + nk:])
    dx, dw = lin.vjp(x, got)
    rx, mx, rw, mw = of.vjp(f32(x), f32(got), f32(lin.codes), f32(lin.scales))
    near(f64(dx), rx, _tol_gemm(mx, lin.N, torch.bfloat16, rx), "dx")
    near(f64(dw), rw, _tol_gemm(mw, T, torch.float32, rw), "dw")
    g = residual_norm_vjp(v["h"], v["y"], v["w_post"], v["w_pre"], st, v["dh"], dx, gate=v["gate"],
                          scale=0.7)
    _check_norm_vjp(dict(v, dx=dx), g, v["dh"], 0.7, 1e-6, 0.0)
    # and the same through the helper that the graphs' test replays
    again = _backward(*args, st, x, dqkv[:, :nq].reshape(T, heads, hd),
                      dqkv[:, nq:nq + nk].reshape(T, kv, hd), dqkv[:, nq + nk:])
    assert all(torch.equal(again[n], w) for n, w in dict(g, dx=dx, dw=dw).items())
    _err_ok()


def test_captured_graphs_streams_and_overlapping_calls():
    """Two graphs of the same objects replayed in turn and on two streams at once give what eager
    calls give; so does a call on a side stream."""
    argsA, argsB = _block(0), _block(50)
    v = argsA[2]

    def step(a):
        h2, x, st, qkv, qr, kr = _forward(*a, fp8=False)
        g = _backward(*a, st, x, qr, kr, a[2]["dx"][:, 128:])
        return [h2, x, st, qkv, qr, kr] + list(g.values())

    # one weight and plan, two inputs
    argsB = (argsA[0], argsA[1], argsB[2], *argsA[3:])
    eager = [step(a) for a in (argsA, argsB)]
    graphs, outs = [], []
    for a in (argsA, argsB):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step(a)
        torch.cuda.current_stream().wait_stream(s)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(step(a))
        graphs.append(gr)
    for _ in range(2):
        for gr in graphs:
            gr.replay()
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for o in outs:
        for t in o:
            t.zero_()
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(s1):
            graphs[0].replay()
        with torch.cuda.stream(s2):
            graphs[1].replay()
    torch.cuda.synchronize()
    for o, e in zip(outs, eager):
        assert all(torch.equal(a, b) for a, b in zip(o, e))
    # eager calls on two streams at once
    with torch.cuda.stream(s1):
        r1 = step(argsA)
    with torch.cuda.stream(s2):
        r2 = step(argsB)
    torch.cuda.synchronize()
    for o, e in zip((r1, r2), eager):
        assert all(torch.equal(a, b) for a, b in zip(o, e))
    _err_ok()


def test_norm_gradients_from_two_host_threads(monkeypatch):
    """Two widths of one kernel that need different amounts of shared memory (82 and 131 KB), called
    by two threads at once: the limit that one sets must not fall below what the other launches.
    The threads repeat the entry point's calls alone, so that they meet in it often."""
    import threading
    from gsq_rco_mlx_b200 import _lib
    from gsq_rco_mlx_b200.common.norm import residual_norm, residual_norm_vjp
    jobs, seen, status = [], [], [[], []]
    real = _lib.call

    def call(name, *args):
        seen.append((name, args))
        real(name, *args)

    for H in (2560, 4096):
        v = _norm_inputs(8, H, "bf16", True, True, 0, H)
        st = residual_norm(v["h"], v["y"], v["w_post"], v["w_pre"])[2]
        side = torch.cuda.Stream()
        with monkeypatch.context() as m, torch.cuda.stream(side):
            side.wait_stream(torch.cuda.default_stream())
            m.setattr(_lib, "call", call)
            got = residual_norm_vjp(v["h"], v["y"], v["w_post"], v["w_pre"], st, v["dh"], v["dx"])
        torch.cuda.synchronize()
        name, args = seen.pop()
        assert name == "gsq_residual_norm_bwd"
        ws = torch.empty(args[-3], device="cuda", dtype=torch.uint8)
        args = args[:-4] + (ws.data_ptr(),) + args[-3:]
        jobs.append((args, got, {n: t.clone() for n, t in got.items() if t is not None},
                     (v, st, ws, side)))
    fn = _lib.lib().gsq_residual_norm_bwd
    start = threading.Barrier(len(jobs))

    def work(i):
        start.wait(30)
        status[i] = [n for n in (fn(*jobs[i][0]) for _ in range(20000)) if n]

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert status == [[], []]
    for _, got, want, _ in jobs:
        assert all(torch.equal(got[n], want[n]) for n in want)
    _err_ok()


def test_residual_norm_refuses_outputs_across_its_inputs():
    from gsq_rco_mlx_b200.common.norm import residual_norm
    buf = rnd((9, 64), 5, torch.bfloat16)
    h, y = buf[:8, :24], buf[:8, 32:56]
    want = residual_norm(h, y)[0]
    for out in (buf[1:, :24], buf[:8, 8:32], buf[1:, 32:56], buf[:8, 40:64],
                buf.flatten()[:8 * 24].view(8, 24)):
        with pytest.raises(ValueError, match="overlaps"):
            residual_norm(h, y, out=out)
    over = h.clone()
    assert torch.equal(residual_norm(over, y, out=over)[0], want)
    over = y.clone()
    assert torch.equal(residual_norm(h, over, out=over)[0], want)
    wide = buf.clone()
    assert torch.equal(residual_norm(wide[:8, :24], wide[:8, 24:48], out=wide[:8, 24:48])[0],
                       residual_norm(h, buf[:8, 24:48])[0])


def test_outputs_over_operands_that_are_still_read():
    """The 8-bit product into its own codes or scales, both gradients in one place, h' over the
    norm's parameters: refused, with nothing written. Into the dense rows that were quantized
    before: the values of a fresh output."""
    from gsq_rco_mlx_b200.common.fp8 import Fp8Linear, quantize_rows
    from gsq_rco_mlx_b200.common.norm import residual_norm
    n = 256
    lin = Fp8Linear.from_weight(rnd((n, n), 1), transposed=True)
    x, dy = rnd((n, n), 2), rnd((n, n), 3)
    q = quantize_rows(x)
    room = q.codes.view(torch.bfloat16)   # [n, n / 2] over the codes
    small = Fp8Linear.from_weight(rnd((n // 2, n), 4))
    keep = q.codes.view(torch.uint8).clone(), q.scales.clone()
    with pytest.raises(ValueError, match="codes of x"):
        small(q, out=room)
    with pytest.raises(ValueError, match="scales of x"):   # (2 blocks of n scales: n rows of two)
        Fp8Linear.from_weight(rnd((2, n), 5))(q, out=q.scales.t().view(n, 2), y_f32=True)
    g = torch.zeros(2 * n, n, device="cuda")
    for a, b in ((g[:n], g[:n]), (g[:n], g[n - 1:2 * n - 1])):
        with pytest.raises(ValueError, match="dx overlaps dw"):
            lin.vjp(x, dy, dx=a, dw=b)
    assert not bool(g.any())
    want = lin.vjp(x, dy)
    got = lin.vjp(x, dy, dx=g[:n], dw=g[n:])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    y = lin(x)
    over = x.clone()
    assert torch.equal(lin(over, out=over), y)
    over = x.clone()
    got = lin.vjp(over, dy, dx=over)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    buf = rnd((9, 64), 6)
    h, z = rnd((8, 64), 7), rnd((8, 64), 8)
    before = buf.clone()
    for kw in ({"w_post": buf[3]}, {"w_pre": buf[0]}, {"gate": buf[4:6]}):
        with pytest.raises(ValueError, match="out overlaps " + next(iter(kw))):
            residual_norm(h, z, out=buf[:8], **kw)
        residual_norm(h, z, out=buf.clone()[:8], **kw)
    assert torch.equal(buf, before)
    assert torch.equal(q.codes.view(torch.uint8), keep[0]) and torch.equal(q.scales, keep[1])
    residual_norm(h, z, w_post=buf[8], out=buf[:8])
    _err_ok()


def test_transposed_codes_are_there_for_every_stream():
    """A weight's first vjp behind other work of its stream, the second at once on another one; and
    a capture that would have to make the codes is refused, with eager calls as right after it."""
    from gsq_rco_mlx_b200.common.fp8 import Fp8Linear
    W, x, dy = rnd((640, 512), 1, torch.bfloat16), rnd((96, 512), 2, torch.bfloat16), \
        rnd((96, 640), 3, torch.bfloat16)
    want = Fp8Linear.from_weight(W, transposed=True).vjp(x, dy)
    lin = Fp8Linear.from_weight(W)
    busy = torch.zeros(1 << 28, device="cuda")
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s1):
        for _ in range(20):
            busy.add_(1.0)
        a = lin.vjp(x, dy)
    with torch.cuda.stream(s2):
        b = lin.vjp(x, dy)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for g in (a, b) for p, q in zip(g, want))
    lin = Fp8Linear.from_weight(W)
    with pytest.raises(RuntimeError, match="before it"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            lin.vjp(x, dy)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(lin.vjp(x, dy), want))
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        c = lin.vjp(x, dy)
    gr.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(c, want))
    _err_ok()


def test_the_error_word_is_there_for_every_stream(monkeypatch):
    """The device's first call behind other work of its stream, over a block that was left nonzero,
    and one on another stream at once: the word that both share is zero for both."""
    from gsq_rco_mlx_b200 import gemm
    from gsq_rco_mlx_b200.common.fp8 import Fp8Linear
    W, x = rnd((640, 512), 1, torch.bfloat16), rnd((96, 512), 2, torch.bfloat16)
    want = Fp8Linear.from_weight(W)(x)
    busy = torch.zeros(1 << 28, device="cuda")
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    monkeypatch.setattr(gemm, "_ERR", {})
    with torch.cuda.stream(s1):
        for n in (1, 8, 64):
            torch.full((n,), 77, device="cuda", dtype=torch.int32)   # left in s1's pool
    torch.cuda.synchronize()
    with torch.cuda.stream(s1):
        for _ in range(20):
            busy.add_(1.0)
        a = Fp8Linear.from_weight(W)(x)
    with torch.cuda.stream(s2):
        first = gemm.err_flag(x.device).clone()
        b = Fp8Linear.from_weight(W)(x)
    torch.cuda.synchronize()
    assert int(first) == 0 and len(gemm._ERR) == 1
    assert torch.equal(a, want) and torch.equal(b, want)
    _err_ok()


def test_fp8_layers_in_the_packed_eval():
    """PackedModel takes Fp8Linear layers: its scratch weights are their dequantized values, and
    the perplexity is that of the dense model with those weights."""
    from gsq_rco_mlx_b200.common.evaluate import PackedModel, perplexity
    from gsq_rco_mlx_b200.common.fp8 import Fp8Linear
    from gsq_rco_mlx_b200.gsq.e2e import LIN_ORDER, BlockConfig
    cfg = BlockConfig(hidden=128, n_heads=2, n_kv=1, head_dim=64, inter=256)
    shapes = {"q_proj": (128, 128), "k_proj": (64, 128), "v_proj": (64, 128), "o_proj": (128, 128),
              "gate_proj": (256, 128), "up_proj": (256, 128), "down_proj": (128, 256)}
    bf = torch.bfloat16
    layers, layers16 = [], []
    for L in range(2):
        d = {"q_bias": rnd((128,), 100 + L, bf, 0.1), "k_bias": rnd((64,), 110 + L, bf, 0.1),
             "v_bias": rnd((64,), 120 + L, bf, 0.1),
             "in_norm": torch.ones(128, device="cuda", dtype=bf),
             "post_norm": torch.ones(128, device="cuda", dtype=bf)}
        d16 = dict(d)
        for i, name in enumerate(LIN_ORDER):
            d[name] = rnd(shapes[name], 10 * L + i, bf, 0.08)
            d16[name] = torch.empty(shapes[name], device="cuda", dtype=bf)
            Fp8Linear.from_weight(d[name]).dequant(d16[name])
        layers.append(d)
        layers16.append(d16)
    embed, nw = rnd((512, 128), 200, bf), torch.ones(128, device="cuda", dtype=bf)
    win = np.random.default_rng(0).integers(0, 512, (3, 128))
    m8 = PackedModel.from_fp8(SimpleNamespace(cfg=cfg, embed=embed, norm=nw, layers=layers))
    m16 = PackedModel(cfg, embed, nw, layers16)
    a, b = perplexity(m8, win), perplexity(m16, win)
    assert a == b and np.isfinite(a["ppl"])
    n = sum(r * c + 4 * -(-r // 128) * -(-c // 128) for r, c in shapes.values())
    assert m8.packed_bytes() == 2 * n and m16.packed_bytes() == 0
    some = PackedModel.from_fp8(SimpleNamespace(cfg=cfg, embed=embed, norm=nw, layers=layers),
                                names=("up_proj",))
    assert some.packed_bytes() == 2 * (256 * 128 + 4 * 2) and some.layers[0]["q_proj"] is \
        layers[0]["q_proj"]
