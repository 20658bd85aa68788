"""Linears in 8-bit floating point: e4m3 values with a float32 scale per block of 128.

Half the bytes of bf16, both operands of the product in 8 bits on the tensor cores, no
calibration. The packed eval takes the weight format beside PackedLinear (common/evaluate.py): it
dequantizes the weights, and its products run on bf16 activations. With a the largest magnitude of
a block and a' = max(a, 2^-100),

  scale = a' / 448,  code = e4m3(x * (448 / a'))        (448: the largest e4m3 value)

  Fp8Tensor      rows of activations: codes [R, C] and a scale per row and 128 columns
  quantize_rows  x -> Fp8Tensor
  Fp8Linear      a weight [N, K] with a scale per 128 x 128: y = x W^T with x quantized in rows,
                 and its vector-Jacobian product

Rows up to 2^30; 65535 blocks of 128 (8.4e6) where they are a weight's, or are quantized by columns
(vjp).

Reference: none (src/gsq_rco/gsq/export.py:52-91 exports integer codes only).
"""
from __future__ import annotations

import torch

from .. import _lib
from .operands import DTYPES, MAX_DIM, apart, error_word, matrix, on_device, output, \
    same_device, stream_of

BLOCK = 128
E4M3 = torch.float8_e4m3fn


def _blocks(n):
    return -(-n // BLOCK)


def pad16(n):
    return -(-n // 16) * 16


class Fp8Tensor:
    """Activations [R, C] in e4m3: codes float8_e4m3fn [R, C] (a view of rows padded to 16
    bytes) and scales float32 [R, ceil(C / 128)] (a view: stored block-major, as the product
    reads them)."""

    def __init__(self, codes, scales):
        R, C = codes.shape
        if R > MAX_DIM or C > MAX_DIM:
            raise ValueError(f"codes have more than {MAX_DIM} rows or columns: {(R, C)}")
        if codes.dtype != E4M3 or scales.dtype != torch.float32:
            raise ValueError("codes must be float8_e4m3fn and scales float32")
        if tuple(scales.shape) != (R, _blocks(C)):
            raise ValueError(f"scales must be [{R}, {_blocks(C)}], got {tuple(scales.shape)}")
        same_device(scales, "scales", on_device(codes, "codes"))
        if R and (C > 1 and codes.stride(1) != 1 or R > 1 and codes.stride(0) < C or
                  codes.stride(0) % 16 or codes.data_ptr() % 16):
            raise ValueError("codes rows must be contiguous with a pitch of a multiple of 16")
        if R > 1 and scales.stride(0) != 1 or scales.shape[1] > 1 and scales.stride(1) < R:
            raise ValueError("scales must be stored block-major ([blocks, rows] transposed)")
        self.codes, self.scales = codes, scales
        self.shape = (R, C)

    @classmethod
    def empty(cls, R, C, dev):
        """Room for [R, C] (built by its own layout: nothing to check)."""
        q = cls.__new__(cls)
        codes = torch.empty(R, pad16(C), device=dev, dtype=E4M3)
        q.codes = codes if C == codes.shape[1] else codes[:, :C]
        q.scales = torch.empty(_blocks(C), R, device=dev, dtype=torch.float32).t()
        q.shape = (R, C)
        return q

    def float(self):
        """The float32 values that the codes stand for."""
        s = self.scales.repeat_interleave(BLOCK, 1)[:, :self.shape[1]]
        return self.codes.float() * s


def quantize_rows(x) -> Fp8Tensor:
    """x [R, C] (bf16, float16 or float32) in e4m3 with a scale per row and 128 columns."""
    x, ld = matrix(x, "x")
    dev = on_device(x, "x")
    R, C = x.shape
    q = Fp8Tensor.empty(R, C, x.device)
    if R and C:
        _lib.call("gsq_fp8_quant", x.data_ptr(), DTYPES[x.dtype], R, C, ld, q.codes.data_ptr(),
                  pad16(C), q.scales.data_ptr(), R, None, 0, None, 0, stream_of(dev))
    return q


def _padded(codes):
    """codes [R, C] with rows on 16 bytes (a copy where they are not)."""
    R, C = codes.shape
    if codes.stride(1) == 1 and codes.stride(0) % 16 == 0 and codes.stride(0) >= C \
            and codes.data_ptr() % 16 == 0:
        return codes
    out = torch.zeros(R, pad16(C), device=codes.device, dtype=torch.uint8)
    out[:, :C].copy_(codes.view(torch.uint8))
    return out.view(E4M3)[:, :C]


class Fp8Linear:
    """One linear W [N, K] in e4m3: codes float8_e4m3fn [N, K], scales float32
    [ceil(N / 128), ceil(K / 128)], both kept as they are where the codes' rows lie on 16 bytes
    (copied otherwise). codes_t: the codes transposed [K, N], which the vector-Jacobian product
    reads (made on its first use otherwise, and not while a graph is captured). The codes are not
    to be written to afterwards."""

    def __init__(self, codes, scales, codes_t=None):
        if codes.dtype != E4M3 or codes.dim() != 2 or not codes.numel():
            raise ValueError(f"codes must be a float8_e4m3fn matrix, got {codes.dtype} "
                             f"{tuple(codes.shape)}")
        self.N, self.K = int(codes.shape[0]), int(codes.shape[1])
        if self.N > MAX_DIM or self.K > MAX_DIM:
            raise ValueError(f"codes have more than {MAX_DIM} rows or columns: "
                             f"{tuple(codes.shape)}")
        if scales.dtype != torch.float32 or \
                tuple(scales.shape) != (_blocks(self.N), _blocks(self.K)):
            raise ValueError(f"scales must be float32 [{_blocks(self.N)}, {_blocks(self.K)}], "
                             f"got {scales.dtype} {tuple(scales.shape)}")
        self.dev = on_device(codes, "codes")
        same_device(scales, "scales", self.dev)
        self.codes, self.scales = _padded(codes), scales.contiguous()
        self._t = None
        if codes_t is not None:
            if codes_t.dtype != E4M3 or tuple(codes_t.shape) != (self.K, self.N):
                raise ValueError(f"codes_t must be float8_e4m3fn [{self.K}, {self.N}]")
            same_device(codes_t, "codes_t", self.dev)
            self._t = _padded(codes_t)
        self._err = error_word(codes.device)
        self._width = pad16(self.K) + 4 * _blocks(self.K)   # workspace bytes of a row

    @classmethod
    def from_weight(cls, W, transposed=False):
        """Quantize a dense weight [N, K] (bf16, float16 or float32); transposed: also keep the
        codes transposed, for vjp."""
        W, ld = matrix(W, "W")
        dev = on_device(W, "W")
        N, K = W.shape
        if not N or not K:
            raise ValueError("W must not be empty")
        codes = torch.empty(N, pad16(K), device=W.device, dtype=E4M3)
        scales = torch.empty(_blocks(N), _blocks(K), device=W.device, dtype=torch.float32)
        _lib.call("gsq_fp8_quant_blocks", W.data_ptr(), DTYPES[W.dtype], N, K, ld,
                  codes.data_ptr(), pad16(K), scales.data_ptr(), _blocks(K), stream_of(dev))
        lin = cls(codes[:, :K], scales)
        if transposed:
            lin.codes_t()
        return lin

    def codes_t(self):
        """The codes transposed [K, N]."""
        if self._t is None:
            if torch.cuda.is_current_stream_capturing():
                # they would be written at the graph's replays only, and read by every call
                raise RuntimeError("the transposed codes cannot be made during a graph capture: "
                                   "call codes_t() before it")
            t = torch.zeros(self.K, pad16(self.N), device=self.codes.device, dtype=torch.uint8)
            t[:, :self.N].copy_(self.codes.view(torch.uint8).t())
            # the next call may come on any stream (once a weight)
            torch.cuda.current_stream(self.dev).synchronize()
            self._t = t.view(E4M3)[:, :self.N]
        return self._t

    def dequant(self, out):
        """out [N, K] (bf16, float16 or float32; rows may be strided) = the dense weight."""
        if out.dtype not in DTYPES:
            raise ValueError(f"unsupported out dtype {out.dtype}")
        dev = on_device(self.codes, "the weight")
        _, ld = output(out, self.N, self.K, out.dtype, self.codes, "out")
        _lib.call("gsq_fp8_dequant", self.codes.data_ptr(), self.codes.stride(0),
                  self.scales.data_ptr(), self.scales.shape[1], self.N, self.K, out.data_ptr(),
                  DTYPES[out.dtype], ld, stream_of(dev))
        return out

    def __call__(self, x, out=None, y_f32=False):
        """y = x W^T [M, N] in x's type (or float32): x [M, K] (bf16, float16 or float32),
        quantized per row and 128 columns on the way (out may lie over it); or x an Fp8Tensor (y in
        bf16, an out over it is refused)."""
        dev = on_device(self.codes, "the weight")
        if isinstance(x, Fp8Tensor):
            M = x.shape[0]
            if x.shape[1] != self.K:
                raise ValueError(f"x must be [M, {self.K}], got {x.shape}")
            same_device(x.codes, "x", dev)
            y, ld = output(out, M, self.N, torch.float32 if y_f32 else torch.bfloat16,
                           self.codes, "out")
            if out is not None:
                apart(out, "out", x.codes, "the codes of x")
                apart(out, "out", x.scales.t(), "the scales of x")
            if M:
                _lib.call("gsq_fp8_gemm", M, self.N, self.K, x.codes.data_ptr(), x.codes.stride(0),
                          x.scales.data_ptr(), x.scales.stride(1) if x.scales.shape[1] > 1 else M,
                          self.codes.data_ptr(), self.codes.stride(0),
                          self.scales.data_ptr(), 0, self.scales.shape[1], 1, y.data_ptr(),
                          DTYPES[y.dtype], ld, 0, self._err.data_ptr(), stream_of(dev))
            return y
        x, ld_x = matrix(x, "x", cols=self.K)
        same_device(x, "x", dev)
        M = x.shape[0]
        y, ld = output(out, M, self.N, torch.float32 if y_f32 else x.dtype, x, "out")
        if not M:
            return y
        # allocated per call on the calling stream: nothing is shared between calls
        nbytes = M * self._width
        ws = x.new_empty((nbytes,), dtype=torch.uint8)
        _lib.call("gsq_fp8_linear", x.data_ptr(), DTYPES[x.dtype], M, self.K, ld_x,
                  self.codes.data_ptr(), self.codes.stride(0), self.scales.data_ptr(),
                  self.scales.shape[1], self.N, y.data_ptr(), DTYPES[y.dtype], ld, ws.data_ptr(),
                  nbytes, self._err.data_ptr(), stream_of(dev))
        return y

    def vjp(self, x, dy, dx=None, dw=None, accumulate=False):
        """Vector-Jacobian product at x [M, K] for the cotangent dy [M, N]: (dx, dw).
        dx = dy W [M, K] in x's type, dy quantized per row and 128 columns, W the weight's own
        codes. dw = dy^T x float32 [N, K] (added to dw when accumulate), both quantized per
        column and 128 rows; rounding counts as the identity (straight through). dx and dw may lie
        over x and dy, but not over one another."""
        if isinstance(x, Fp8Tensor):
            raise ValueError("x must be dense: dw takes it with other scales (per column and 128 "
                             "rows) than the rows' codes hold")
        dev = on_device(self.codes, "the weight")
        x, ld_x = matrix(x, "x", cols=self.K)
        M, N, K = x.shape[0], self.N, self.K
        dy, ld_dy = matrix(dy, "dy", rows=M, cols=N)
        same_device(x, "x", dev)
        same_device(dy, "dy", dev)
        if accumulate and dw is None:
            raise ValueError("accumulate needs dw")
        both = dx is not None and dw is not None
        dx, ld_dx = output(dx, M, K, x.dtype, x, "dx")
        dw, ld_dw = output(dw, N, K, torch.float32, x, "dw")
        if both:
            apart(dx, "dx", dw, "dw")
        if not M:
            if not accumulate:
                dw.zero_()
            return dx, dw
        wt = self.codes_t()
        nbytes = M * pad16(N) + (N + K) * pad16(M) + 4 * (M * _blocks(N) + (N + K) * _blocks(M))
        # allocated per call on the calling stream: nothing is shared between calls
        ws = x.new_empty((nbytes,), dtype=torch.uint8)
        _lib.call("gsq_fp8_linear_vjp", x.data_ptr(), DTYPES[x.dtype], M, K, ld_x, dy.data_ptr(),
                  DTYPES[dy.dtype], N, ld_dy, wt.data_ptr(), wt.stride(0), self.scales.data_ptr(),
                  self.scales.shape[1], dx.data_ptr(), ld_dx, dw.data_ptr(), ld_dw, accumulate,
                  ws.data_ptr(), nbytes, self._err.data_ptr(), stream_of(dev))
        return dx, dw
