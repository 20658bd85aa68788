// Element types of the operators that take bf16, float16 or float32 (0, 1, 2 in the C ABI), and
// vectors of eight of them.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace gsq {

// Rows and columns that a launch takes: 32-bit counts plus a grid's step stay in range.
constexpr int kMaxDim = 1 << 30;

enum DType { BF16 = 0, F16 = 1, F32 = 2 };

inline size_t dtype_size(int dtype) { return dtype == F32 ? 4 : 2; }

// A pointer that lies on `size` bytes, as the kernels' accesses need it (or is missing).
inline bool lies_on(const void* p, size_t size) { return (uintptr_t)p % size == 0; }

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// Pairs of float32 in one instruction (each half rounds as the scalar operation does): the fused
// multiply-add of a pair issues as fast as a single one.
struct F2 {
  uint64_t b;   // held as the packed operations take it: a pair of registers, not two
  F2() = default;
  __device__ __forceinline__ F2(float x, float y) {
    asm("mov.b64 %0, {%1, %2};" : "=l"(b) : "f"(x), "f"(y));
  }
  __device__ __forceinline__ explicit F2(uint64_t bits) : b(bits) {}
  __device__ __forceinline__ float x() const { return __uint_as_float((uint32_t)b); }
  __device__ __forceinline__ float y() const { return __uint_as_float((uint32_t)(b >> 32)); }
};
__device__ __forceinline__ F2 f2_fma(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.b) : "l"(a.b), "l"(b.b), "l"(c.b));
  return r;
}
__device__ __forceinline__ F2 f2_mul(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.b) : "l"(a.b), "l"(b.b));
  return r;
}
__device__ __forceinline__ F2 f2_add(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.b) : "l"(a.b), "l"(b.b));
  return r;
}
__device__ __forceinline__ F2 f2_same(float v) { return {v, v}; }

// Two neighbouring 16-bit values (one word) as a pair, and back.
template <typename T>
__device__ __forceinline__ F2 f2_unpack(uint32_t w);
template <>
__device__ __forceinline__ F2 f2_unpack<__nv_bfloat16>(uint32_t w) {
  return {__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)};
}
template <>
__device__ __forceinline__ F2 f2_unpack<__half>(uint32_t w) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  return {f.x, f.y};
}
template <typename T>
__device__ __forceinline__ uint32_t f2_pack(F2 v);
template <>
__device__ __forceinline__ uint32_t f2_pack<__nv_bfloat16>(F2 v) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(v.x(), v.y());
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t f2_pack<__half>(F2 v) {
  const __half2 h = __floats2half2_rn(v.x(), v.y());
  return *reinterpret_cast<const uint32_t*>(&h);
}

// A row's columns are dealt to a team of tpr threads in fours: column j < 4 of a thread's chunk q
// is one of four neighbours (VEC: chunks go round the team; a warp's chunk is 128 columns), or
// goes round the team by itself, which keeps every access of a warp to a row one segment.
template <bool VEC>
__device__ __forceinline__ int column(int q, int j, int t, int tpr) {
  return VEC ? (q * tpr + t) * 4 + j : (q * 4 + j) * tpr + t;
}

// Chunk q of a row as it lies in memory; columns from H on are zero. VEC: H is a multiple of 4
// and the row starts on 8 (16-bit types) or 16 bytes. PAD: the row has room for the whole team's
// columns, so it may be read past H.
template <typename T>
struct alignas(4 * sizeof(T)) Four {
  T e[4];
};

template <typename T, bool VEC, bool PAD>
__device__ __forceinline__ Four<T> raw4(const T* row, int q, int t, int tpr, int H) {
  const int c0 = column<VEC>(q, 0, t, tpr);
  Four<T> v;
  if constexpr (VEC) {
    if constexpr (sizeof(T) == 2) {
      uint2 r = make_uint2(0u, 0u);
      if (c0 < H) r = *reinterpret_cast<const uint2*>(row + c0);
      *reinterpret_cast<uint2*>(&v) = r;
    } else {
      float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
      if (c0 < H) r = *reinterpret_cast<const float4*>(row + c0);
      *reinterpret_cast<float4*>(&v) = r;
    }
  } else {
    const T zero = from_f32<T>(0.f);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int col = c0 + j * tpr;
      if (PAD) {
        v.e[j] = row[col];
        v.e[j] = col < H ? v.e[j] : zero;
      } else {
        v.e[j] = col < H ? row[col] : zero;
      }
    }
  }
  return v;
}

// The chunk's values as two pairs (VEC: unpacked a word at a time).
template <typename T, bool VEC>
__device__ __forceinline__ void pairs(const Four<T>& r, F2 v[2]) {
  if constexpr (VEC && sizeof(T) == 2) {
    const uint2 w = *reinterpret_cast<const uint2*>(&r);
    v[0] = f2_unpack<T>(w.x);
    v[1] = f2_unpack<T>(w.y);
  } else {
    v[0] = {to_f32(r.e[0]), to_f32(r.e[1])};
    v[1] = {to_f32(r.e[2]), to_f32(r.e[3])};
  }
}

// maximum that keeps NaN (fmaxf drops it)
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// e4m3 blocks of 128 values: scale = a / 448 and codes e4m3(x (448 / a)) with a the largest
// magnitude, at least 2^-100 (which keeps 448 / a finite for zeros and denormals).
constexpr int kFp8Block = 128;
constexpr float kFp8Max = 448.f;
constexpr float kFp8AmaxMin = 7.8886090522101181e-31f;  // 2^-100

// Bits of the largest magnitude of four (magnitudes compare as their bits, NaN above infinity).
__device__ __forceinline__ uint32_t amax4(const F2 v[2]) {
  return max(max(__float_as_uint(fabsf(v[0].x())), __float_as_uint(fabsf(v[0].y()))),
             max(__float_as_uint(fabsf(v[1].x())), __float_as_uint(fabsf(v[1].y()))));
}

__device__ __forceinline__ uint32_t cvt4_e4m3(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}

__device__ __forceinline__ uint32_t encode4(const F2 v[2], float r) {
  const F2 a = f2_mul(v[0], f2_same(r)), b = f2_mul(v[1], f2_same(r));
  return cvt4_e4m3(a.x(), a.y(), b.x(), b.y());
}

// Writes a chunk's codes (as raw4 deals columns): one word, or a byte each.
template <bool VEC>
__device__ __forceinline__ void put_codes(uint8_t* row, int q, int t, int tpr, int H, uint32_t c) {
  const int c0 = column<VEC>(q, 0, t, tpr);
  if (VEC) {
    if (c0 < H) *reinterpret_cast<uint32_t*>(row + c0) = c;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c0 + j * tpr < H) row[c0 + j * tpr] = (uint8_t)(c >> (8 * j));
  }
}

}  // namespace gsq
