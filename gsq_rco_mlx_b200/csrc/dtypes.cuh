// Element types of the operators that take bf16, float16 or float32 (0, 1, 2 in the C ABI), and
// vectors of eight of them.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace gsq {

enum DType { BF16 = 0, F16 = 1, F32 = 2 };

inline size_t dtype_size(int dtype) { return dtype == F32 ? 4 : 2; }

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

// Eight values of a row from column c on; columns past `cols` are zero. VEC: the row starts on
// 16 bytes and c is a multiple of 8.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* __restrict__ row, int c, int cols, float v[8]) {
  if (VEC && c + 8 <= cols) {
    constexpr int N4 = sizeof(T) * 8 / 16;
    uint4 raw[N4];
#pragma unroll
    for (int i = 0; i < N4; ++i) raw[i] = reinterpret_cast<const uint4*>(row + c)[i];
    const T* e = reinterpret_cast<const T*>(raw);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = to_f32(e[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c + j < cols ? to_f32(row[c + j]) : 0.f;
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* __restrict__ row, int c, int cols, const float v[8]) {
  if (VEC && c + 8 <= cols) {
    constexpr int N4 = sizeof(T) * 8 / 16;
    __align__(16) T e[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) e[j] = from_f32<T>(v[j]);
#pragma unroll
    for (int i = 0; i < N4; ++i)
      reinterpret_cast<uint4*>(row + c)[i] = reinterpret_cast<const uint4*>(e)[i];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j < cols) row[c + j] = from_f32<T>(v[j]);
  }
}

// Pairs of float32 in one instruction (each half rounds as the scalar operation does): the fused
// multiply-add of a pair issues as fast as a single one.
struct F2 {
  float x, y;
};
__device__ __forceinline__ uint64_t f2_bits(F2 v) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.x), "f"(v.y));
  return r;
}
__device__ __forceinline__ F2 f2_of(uint64_t r) {
  F2 v;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(r));
  return v;
}
__device__ __forceinline__ F2 f2_fma(F2 a, F2 b, F2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(f2_bits(a)), "l"(f2_bits(b)), "l"(f2_bits(c)));
  return f2_of(r);
}
__device__ __forceinline__ F2 f2_mul(F2 a, F2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(f2_bits(a)), "l"(f2_bits(b)));
  return f2_of(r);
}
__device__ __forceinline__ F2 f2_add(F2 a, F2 b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(f2_bits(a)), "l"(f2_bits(b)));
  return f2_of(r);
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
  const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t f2_pack<__half>(F2 v) {
  const __half2 h = __floats2half2_rn(v.x, v.y);
  return *reinterpret_cast<const uint32_t*>(&h);
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

__device__ __forceinline__ float amax8(const float v[8]) {
  float a = fabsf(v[0]);
#pragma unroll
  for (int j = 1; j < 8; ++j) a = max_nan(a, fabsf(v[j]));
  return a;
}

__device__ __forceinline__ uint32_t cvt4_e4m3(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}

__device__ __forceinline__ uint2 encode8(const float v[8], float r) {
  float q[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) q[j] = __fmul_rn(v[j], r);
  return make_uint2(cvt4_e4m3(q[0], q[1], q[2], q[3]), cvt4_e4m3(q[4], q[5], q[6], q[7]));
}

}  // namespace gsq
