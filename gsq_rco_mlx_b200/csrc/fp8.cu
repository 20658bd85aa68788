// Products of e4m3 matrices with a float32 scale per block of 128 values.
//
// A matrix X [R][C] is held as e4m3 codes and scales: per row and 128 consecutive columns
// ("rows", the activations), or per 128 x 128 ("blocks", the weights). With a the largest
// magnitude of a block, a' = max(a, 2^-100):
//   scale = a' / 448, code = e4m3(x * (448 / a'))        (float32, each operation rounded once)
// 448 is the largest e4m3 value, so the largest value of a block always lands on it; the floor
// keeps 448 / a' finite for blocks of zeros and of denormals. NaN or infinity in a block make
// its values NaN.
//
// The product: C[m][n] = sum_b sa[b][m] sb(b, n) sum_{k in block b} A[m][k] B[n][k].
// The inner sums run on the tensor cores (kind::f8f6f4: exact products, float32 accumulators in
// TMEM), one accumulator per 128-wide k-block. The scales differ from block to block, so an
// accumulator cannot run on over k: the epilogue warps read it back, and fold it into float32
// registers with one multiply-add per value, two values an instruction.
//
// What bounds it: at the e4m3 rate a 128 x 256 tile takes 512 cycles per k-block. 8191 x 8192 x 4096
// on B200 takes 253 us in bursts at 1965 MHz (2.2 PFLOP/s, the tensor pipe active on 55 % of the
// cycles in a profile), about 1100 cycles each; run for a second, at the 1550 MHz that the power cap
// leaves, 295 us. The fold of a k-block takes 128 packed multiply-adds on each of the four
// schedulers, measured alone at 2.2 cycles each with two warps and 5.4 with one, and the polls of
// barriers, the reads of TMEM and the waits between leave a warp alone for part of the time. Tried
// and dropped: 16 epilogue warps (327 against 296 us), the next columns read while these are folded
// (321 against 285). The loops of the other warps have to stay shorter than the fold: run by one
// lane, the MMA warp's took 840 cycles a k-block, so its control is uniform over the warp.
#include <cuda_fp8.h>

#include <type_traits>

#include "dtypes.cuh"
#include "tc_common.cuh"

namespace gsq {
namespace fp8 {

constexpr int kBlk = kFp8Block;

// ---------------------------------------------------------------------- quantization ---
// Magnitudes of a chunk as bits that compare as they do: 16-bit types two to a word.
template <typename T>
struct Mags {
  static constexpr int N = sizeof(T) == 2 ? 2 : 4;
  uint32_t w[N];
};

template <typename T>
__device__ __forceinline__ Mags<T> mags(const Four<T>& r) {
  Mags<T> m;
  if constexpr (sizeof(T) == 2) {
    const uint2 u = *reinterpret_cast<const uint2*>(&r);
    m.w[0] = u.x & 0x7fff7fffu;
    m.w[1] = u.y & 0x7fff7fffu;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) m.w[j] = __float_as_uint(r.e[j]) & 0x7fffffffu;
  }
  return m;
}

template <typename T>
__device__ __forceinline__ void mags_max(Mags<T>& a, const Mags<T>& b) {
#pragma unroll
  for (int i = 0; i < Mags<T>::N; ++i)
    a.w[i] = sizeof(T) == 2 ? __vmaxu2(a.w[i], b.w[i]) : max(a.w[i], b.w[i]);
}

// The float32 value of the bits of one magnitude.
template <typename T>
__device__ __forceinline__ float mag_value(uint32_t m) {
  if constexpr (sizeof(T) == 2) {
    const uint16_t h = (uint16_t)m;
    return to_f32(*reinterpret_cast<const T*>(&h));
  } else {
    return __uint_as_float(m);
  }
}

// The warp's largest magnitude (bits).
template <typename T>
__device__ __forceinline__ uint32_t warp_top(const Mags<T>& m) {
  uint32_t v;
  if constexpr (sizeof(T) == 2) {
    const uint32_t w = __vmaxu2(m.w[0], m.w[1]);
    v = max(w & 0xffffu, w >> 16);
  } else {
    v = max(max(m.w[0], m.w[1]), max(m.w[2], m.w[3]));
  }
  return __reduce_max_sync(0xffffffffu, v);
}

// The quotients m / 448 (scale) and 448 / m of N <= 16 blocks with maxima m[i] (bits), in one
// division by the warp: lane 2 i holds the scale of block i, lane 2 i + 1 its reciprocal.
template <typename T, int N>
__device__ __forceinline__ float quotients(const uint32_t m[N], int lane) {
  uint32_t b = 0u;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (lane >> 1 == i) b = m[i];
  const float v = max_nan(mag_value<T>(b), kFp8AmaxMin);
  return __fdiv_rn(lane & 1 ? kFp8Max : v, lane & 1 ? v : kFp8Max);
}

// Eight rows' loads of one 128-column block, or R of them. FULL: the block is whole.
template <typename T, bool VEC, bool FULL, int R>
__device__ __forceinline__ void load_rows(const T* src, int64_t ld, int rows, int H, int lane,
                                          Four<T> raw[R]) {
#pragma unroll
  for (int i = 0; i < R; ++i) {
    raw[i] = raw4<T, VEC, false>(src, 0, lane, 32, FULL ? kBlk : (i < rows ? H : 0));
    if (FULL || i + 1 < rows) src += ld;
  }
}

// R rows' codes in row form, and their scales (lanes 2 i).
template <typename T, bool VEC, bool FULL, int R>
__device__ __forceinline__ void put_rows(const Four<T> raw[R], const uint32_t m[R], int rows, int H,
                                         int lane, uint8_t* dst, int64_t ld_c, float* scales) {
  const float quot = quotients<T, R>(m, lane);
  if ((lane & 1) == 0 && lane < 2 * R && (FULL || (lane >> 1) < rows)) scales[lane >> 1] = quot;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    F2 v[2];
    pairs<T, VEC>(raw[i], v);
    const float r = __shfl_sync(0xffffffffu, quot, 2 * i + 1);
    if (FULL || i < rows) put_codes<VEC>(dst, 0, lane, 32, FULL ? kBlk : H, encode4(v, r));
    dst += ld_c;
  }
}

// Rows: a warp takes eight rows of one 128-column block, four columns a lane (a row's maximum is
// one warp reduction, the eight scales are neighbours). One pass over x, eight rows' loads in
// flight: bound by its bytes (8191 x 4096 float16: 19 us, 5.3 TB/s).
constexpr int kRowsWarp = 8;
template <typename T, bool VEC>
__global__ void __launch_bounds__(256, 4)
quant_rows_kernel(const T* __restrict__ x, int64_t ld_x, int rows, int cols, int nblk,
                  uint8_t* __restrict__ codes, int64_t ld_c, float* __restrict__ scales,
                  int64_t ld_s) {
  // (a product launched on these rows may set itself up while they are made)
  asm volatile("griddepcontrol.launch_dependents;");
  const int lane = threadIdx.x & 31;
  const int64_t items = (int64_t)((rows + kRowsWarp - 1) / kRowsWarp) * nblk;
  const int64_t warps = (int64_t)gridDim.x * 8;
  for (int64_t it = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); it < items; it += warps) {
    const int rg = (int)(it / nblk), b = (int)(it - (int64_t)rg * nblk);
    const int r0 = rg * kRowsWarp, H = cols - b * kBlk, left = rows - r0;
    const T* src = x + (int64_t)r0 * ld_x + b * kBlk;
    uint8_t* dst = codes + (int64_t)r0 * ld_c + b * kBlk;
    float* sc = scales + (int64_t)b * ld_s + r0;
    auto work = [&](auto full) {
      constexpr bool FULL = decltype(full)::value;
      Four<T> raw[kRowsWarp];
      load_rows<T, VEC, FULL, kRowsWarp>(src, ld_x, left, H, lane, raw);
      uint32_t m[kRowsWarp];
#pragma unroll
      for (int i = 0; i < kRowsWarp; ++i) m[i] = warp_top<T>(mags(raw[i]));
      put_rows<T, VEC, FULL, kRowsWarp>(raw, m, left, H, lane, dst, ld_c, sc);
    };
    if (H >= kBlk && left >= kRowsWarp) work(std::true_type());
    else work(std::false_type());
  }
}

// A 128 x 128 tile per CTA, sixteen rows a warp and four columns a lane, in any of three forms
// from one read of the tile:
//   ROWS    a scale per row          -> codes [rows][ld_c], scales [cols / 128][ld_s]
//   COLS    a scale per column       -> codes_t [cols][ld_ct], scales_t [rows / 128][ld_st]: a
//           lane's sixteen rows of a column are one 16-byte chunk of the transposed row, swizzled
//           in shared memory so that neither the writes nor the reads of chunks conflict
//   BLOCKS  one scale for the tile   -> codes, scales [rows / 128][ld_s]
// 4094 x 4864 bf16 in rows and columns: 18.5 us, 4.3 TB/s.
template <typename T, bool VEC, bool ROWS, bool COLS, bool BLOCKS>
__global__ void __launch_bounds__(256, sizeof(T) == 2 && (VEC || !ROWS) ? 3 : 2)
quant_tile_kernel(const T* __restrict__ x, int64_t ld_x, int rows, int cols,
                  uint8_t* __restrict__ codes, int64_t ld_c, float* __restrict__ scales,
                  int64_t ld_s, uint8_t* __restrict__ codes_t, int64_t ld_ct,
                  float* __restrict__ scales_t, int64_t ld_st) {
  constexpr int R = 16;
  __shared__ __align__(16) uint32_t red[8][kBlk];
  __shared__ __align__(16) float inv[kBlk];
  __shared__ __align__(16) uint8_t tile[COLS ? kBlk : 1][kBlk];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int cb = blockIdx.x, rb = blockIdx.y;
  const int r0 = rb * kBlk + w * R, H = cols - cb * kBlk, left = rows - r0;
  const T* src = x + (int64_t)(left > 0 ? r0 : 0) * ld_x + cb * kBlk;
  uint8_t* dst = codes + (int64_t)r0 * ld_c + cb * kBlk;
  Four<T> raw[R];
  auto work = [&](auto full) {
    constexpr bool FULL = decltype(full)::value;
    load_rows<T, VEC, FULL, R>(src, ld_x, left, H, lane, raw);
    Mags<T> top = mags(raw[0]);   // the columns' maxima over the warp's rows
    uint32_t m[ROWS ? R : 1];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const Mags<T> a = mags(raw[i]);
      if (ROWS) m[ROWS ? i : 0] = warp_top<T>(a);
      if (i) mags_max(top, a);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      red[w][column<VEC>(0, j, lane, 32)] =
          sizeof(T) == 2 ? (top.w[j >> 1] >> (16 * (j & 1))) & 0xffffu : top.w[sizeof(T) == 2 ? 0 : j];
    if (ROWS)
      put_rows<T, VEC, FULL, ROWS ? R : 1>(raw, m, left, H, lane, dst, ld_c,
                                           scales + (int64_t)cb * ld_s + r0);
  };
  if (H >= kBlk && left >= R) work(std::true_type());
  else work(std::false_type());
  __syncthreads();
  if (COLS) {
    if (threadIdx.x < kBlk) {
      uint32_t a = 0u;
#pragma unroll
      for (int i = 0; i < 8; ++i) a = max(a, red[i][threadIdx.x]);
      const float v = max_nan(mag_value<T>(a), kFp8AmaxMin);
      inv[threadIdx.x] = __fdiv_rn(kFp8Max, v);
      if ((int)threadIdx.x < H)
        scales_t[(int64_t)rb * ld_st + cb * kBlk + threadIdx.x] = __fdiv_rn(v, kFp8Max);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = column<VEC>(0, j, lane, 32);
      const F2 r = f2_same(inv[c]);
      uint32_t q[4];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const Four<T>* f = raw + 4 * g;
        const F2 a = f2_mul(F2(to_f32(f[0].e[j]), to_f32(f[1].e[j])), r),
                 b = f2_mul(F2(to_f32(f[2].e[j]), to_f32(f[3].e[j])), r);
        q[g] = cvt4_e4m3(a.x(), a.y(), b.x(), b.y());
      }
      const int at = w ^ ((VEC ? c >> 2 : c) & 7);
      *reinterpret_cast<uint4*>(&tile[COLS ? c : 0][at * 16]) = make_uint4(q[0], q[1], q[2], q[3]);
    }
    __syncthreads();
#pragma unroll
    for (int e = threadIdx.x; e < kBlk * 8; e += 256) {
      const int c = e >> 3, k = e & 7, at = k ^ ((VEC ? c >> 2 : c) & 7);
      // (the pitch is a multiple of 16: a chunk that holds a row lies inside it)
      if (c < H && rb * kBlk + k * 16 < rows)
        *reinterpret_cast<uint4*>(codes_t + (int64_t)(cb * kBlk + c) * ld_ct + rb * kBlk + k * 16) =
            *reinterpret_cast<const uint4*>(&tile[COLS ? c : 0][at * 16]);
    }
  }
  if (BLOCKS) {
    uint32_t a = 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) a = max(a, red[i][32 * j + lane]);
    a = __reduce_max_sync(0xffffffffu, a);
    const float v = max_nan(mag_value<T>(a), kFp8AmaxMin);
    if (threadIdx.x == 0) scales[(int64_t)rb * ld_s + cb] = __fdiv_rn(v, kFp8Max);
    const float r = __fdiv_rn(kFp8Max, v);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      F2 u[2];
      pairs<T, VEC>(raw[i], u);
      if (i < left) put_codes<VEC>(dst + i * ld_c, 0, lane, 32, H, encode4(u, r));
    }
  }
}

// out = scale[n / 128][k / 128] code, rounded once; eight codes a thread.
template <typename T>
__global__ void __launch_bounds__(256)
dequant_blocks_kernel(const uint8_t* __restrict__ codes, int64_t ld_c,
                      const float* __restrict__ scales, int64_t ld_s, int N, int K,
                      T* __restrict__ out, int64_t ld_o) {
  const int per = (K + 7) / 8;
  const int64_t items = (int64_t)N * per;
  for (int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; e < items;
       e += (int64_t)gridDim.x * blockDim.x) {
    const int n = (int)(e / per), k = (int)(e - (int64_t)n * per) * 8;
    const uint2 raw = *reinterpret_cast<const uint2*>(codes + (int64_t)n * ld_c + k);
    const __nv_fp8_e4m3* q = reinterpret_cast<const __nv_fp8_e4m3*>(&raw);
    const float s = scales[(int64_t)(n / kBlk) * ld_s + k / kBlk];
    T* o = out + (int64_t)n * ld_o + k;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (k + j < K) o[j] = from_f32<T>(__fmul_rn(s, (float)q[j]));
  }
}

// --------------------------------------------------------------------------- product ---
constexpr int kBM = 128;
constexpr int kEpiWarps = 8;
constexpr int kThreads = 128 + 32 * kEpiWarps;
constexpr int kMaxStages = 8;
constexpr uint32_t kPipeBytes = 144 * 1024;
constexpr uint32_t kStageBytes = kEpiWarps * 2 * 4096;  // output boxes, two a warp
constexpr uint32_t kTmemCols = 512;

struct GemmArgs {
  CUtensorMap a, b, o;
  int M, N, K, kb;
  int mt, nt;       // tiles along m and n
  int group;        // m tiles walked together (tile order)
  const float* sa;  // [kb][ld_sa]
  int64_t ld_sa;
  const float* sb;  // blocks: [n / 128][kb] through sb_n, sb_k; rows: [kb][n]
  int64_t sb_n, sb_k;
  void* out;
  int64_t ld_o;
  int accumulate, boxes;  // boxes: out is written through the map o
  int* err;
};

// kind::f8f6f4 instruction descriptor: e4m3 x e4m3 -> float32, both K-major.
constexpr uint32_t idesc_e4m3(int M, int N) {
  return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

template <bool PAIR>
__device__ __forceinline__ void umma_e4m3(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                          uint32_t accumulate) {
  if constexpr (PAIR)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
}

// Arrive on `bar` (PAIR: on the barrier at this address in both CTAs) once the MMAs issued so far
// have completed.
template <bool PAIR>
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
  if constexpr (PAIR)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
        " [%0], %1;" ::"r"(tc::smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
  else
    tc::umma_commit(bar);
}

template <bool PAIR>
__device__ __forceinline__ void tmem_alloc(uint32_t* dst, uint32_t ncols) {
  if constexpr (PAIR) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     tc::smem_u32(dst)),
                 "r"(ncols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  } else {
    tc::tmem_alloc(dst, ncols);
  }
}

template <bool PAIR>
__device__ __forceinline__ void tmem_dealloc(uint32_t taddr, uint32_t ncols) {
  if constexpr (PAIR)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols));
  else
    tc::tmem_dealloc(taddr, ncols);
}

// This shared-memory address in the pair's first CTA.
__device__ __forceinline__ uint32_t leader_u32(const void* ptr) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(tc::smem_u32(ptr)));
  return a;
}

// (What it orders is the reads of TMEM before it, which tcgen05.wait::ld and the fence have
// completed; release.cluster would add a memory barrier of some thousand cycles.)
__device__ __forceinline__ void arrive_leader(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(leader_u32(bar))
               : "memory");
}

// A box into this CTA's shared memory, its bytes counted on the first CTA's barrier.
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, uint32_t bar,
                                                 int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(tc::smem_u32(dst)),
      "l"((uint64_t)map), "r"(bar), "r"(x), "r"(y)
      : "memory");
}

// Until the kernels that this one was launched to follow are complete (no wait otherwise).
__device__ __forceinline__ void grid_wait() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// (.aligned: the warp's threads arrive together, whatever branches they come from)
__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
}

// acc += (d0, d1) s, and acc += ((d0, d1) b) s, on pairs
__device__ __forceinline__ void fold(uint64_t& acc, uint32_t d0, uint32_t d1, uint64_t s) {
  asm("{\n\t.reg .b64 d;\n\tmov.b64 d, {%1, %2};\n\tfma.rn.f32x2 %0, d, %3, %0;\n\t}"
      : "+l"(acc)
      : "r"(d0), "r"(d1), "l"(s));
}
__device__ __forceinline__ void fold2(uint64_t& acc, uint32_t d0, uint32_t d1, uint64_t b,
                                      uint64_t s) {
  asm("{\n\t.reg .b64 d;\n\tmov.b64 d, {%1, %2};\n\tmul.rn.f32x2 d, d, %3;\n\t"
      "fma.rn.f32x2 %0, d, %4, %0;\n\t}"
      : "+l"(acc)
      : "r"(d0), "r"(d1), "l"(b), "l"(s));
}

// Four bytes to shared memory, or zero.
__device__ __forceinline__ void copy4(float* to, const float* from, bool on) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(tc::smem_u32(to)),
               "l"(from), "r"(on ? 4 : 0)
               : "memory");
}

// 64 columns of this thread's lane; no wait.
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, "
      "%18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, "
      "%34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, "
      "%50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63 "
      "}, [%64];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]),
        "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]),
        "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]),
        "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
        "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]),
        "=r"(r[63])
      : "r"(taddr));
}

// The warp's wait for a phase: one poll by all lanes where the phase is there already (control
// stays uniform over the warp, so what follows is issued from uniform registers); bounded as
// tc::mbar_wait.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* err, int code) {
  if (__all_sync(0xffffffffu, tc::mbar_try_wait(bar, parity))) return true;
  const long long t0 = clock64();
  for (uint32_t i = 1;; ++i) {
    if (__all_sync(0xffffffffu, tc::mbar_try_wait(bar, parity))) return true;
    if ((i & 255u) == 0) {
      const bool late = clock64() - t0 > tc::kWaitCycles;
      if (late) atomicCAS(err, 0, code);
      if (__any_sync(0xffffffffu, late || *(volatile int*)err != 0)) return false;
    }
  }
}

__device__ __forceinline__ bool elect_one() {
  uint32_t on;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(on));
  return on != 0;
}

// A place in a ring of N barriers and the parity of its current phase.
template <int N>
struct Turn {
  uint32_t i = 0, phase = 0;
  __device__ __forceinline__ void next() {
    if (++i == N) {
      i = 0;
      phase ^= 1;
    }
  }
};

constexpr int kRing = 8;   // k-blocks whose scales are in shared memory

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(tc::smem_u32(bar)) : "memory");
}

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   (uint64_t)map),
               "r"(tc::smem_u32(src)), "r"(x), "r"(y)
               : "memory");
}

// Tile t in groups of `group` row tiles: within a group the row tile runs fastest, so the CTAs
// in flight share a few row tiles of A and a few column tiles of B in L2.
__device__ __forceinline__ void tile_at(const GemmArgs& p, int t, int& m, int& n) {
  const int per = p.group * p.nt;
  const int g = t / per, i = t - g * per;
  const int rows = min(p.group, p.mt - g * p.group);
  n = i / rows;
  m = g * p.group + (i - n * rows);
}

// An output row's values of one warp column range, element by element (rows that TMA cannot
// write, and sums into what is there): 32 rows an instruction, so an output off 16 bytes costs a
// large product several times its time (16384 x 896 -> 4863: 822 us, -> 4864: 92).
template <typename T, int CW>
__device__ __forceinline__ void store_row(const GemmArgs& p, int m, int n0,
                                          const uint64_t* acc) {
  if (m >= p.M) return;
  T* o = reinterpret_cast<T*>(p.out) + (int64_t)m * p.ld_o + n0;
#pragma unroll
  for (int c = 0; c < CW; ++c) {
    const F2 a(acc[c >> 1]);
    const float v = c & 1 ? a.y() : a.x();
    if (n0 + c < p.N) o[c] = from_f32<T>(p.accumulate ? v + to_f32(o[c]) : v);
  }
}

// The tile's rows of one warp as boxes of 32 rows x 128 bytes, staged in shared memory in the
// store's 128-byte swizzle (16-byte chunk c of row r at c ^ (r % 8): a lane writes its own row
// without bank conflicts) and written by the TMA unit, which clips what lies outside the
// output. Two buffers a warp: a box is written while the last one is still being read.
template <typename T, int CW>
__device__ __forceinline__ void store_boxes(const GemmArgs& p, uint8_t* stage, int& buf, int lane,
                                            int m0, int n0, const uint64_t* acc) {
  constexpr int BW = 128 / sizeof(T);  // columns of a box
  if (m0 >= p.M) return;
#pragma unroll
  for (int c0 = 0; c0 < CW; c0 += BW) {
    if (n0 + c0 < p.N) {
      uint8_t* box = stage + buf * 4096;
      if (lane == 0) tc::bulk_wait_read<1>();
      __syncwarp();
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        uint4 v;
        if constexpr (sizeof(T) == 2) {
          const uint64_t* a = acc + (c0 + c * 8) / 2;
          v = make_uint4(f2_pack<T>(F2(a[0])), f2_pack<T>(F2(a[1])), f2_pack<T>(F2(a[2])),
                         f2_pack<T>(F2(a[3])));
        } else {
          const uint64_t a = acc[(c0 + c * 4) / 2], b = acc[(c0 + c * 4) / 2 + 1];
          v = make_uint4((uint32_t)a, (uint32_t)(a >> 32), (uint32_t)b, (uint32_t)(b >> 32));
        }
        *reinterpret_cast<uint4*>(box + lane * 128 + ((c ^ (lane & 7)) << 4)) = v;
      }
      tc::fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) {
        tma_store_2d(&p.o, box, n0 + c0, m0);
        tc::bulk_commit();
      }
      buf ^= 1;
    }
  }
}

// Register split of the wide kernel: 12 warps are launched with 168 registers a thread; warps
// 0-3 give theirs up to 72 and the epilogue's two warpgroups take 216 (128 x 72 + 256 x 216 =
// 384 x 168): 128 sums and the 64 accumulator columns that are being folded. With a scale per row
// of both sides the columns' scales come on top, and 112 bytes a thread spill (560 read back).
constexpr int kLaunchRegs = 168;
template <int R>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R));
}
template <int R>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R));
}

// Persistent: CTA i takes tiles i, i + gridDim.x, ...  Warp 0 feeds the stages by TMA, warp 1
// issues the MMAs of a k-block into the next accumulator of the ring, warps 4-11 fold it: warp
// w reads TMEM lanes 32 (w % 4).. (its rows) and half of the columns.
// BROWS: B has a scale per row and k-block instead of one per 128 x 128.
// PAIR (256 columns): two CTAs of a cluster share a tile of 256 rows. Each loads its 128 rows of A
// and half of B's columns, the first one issues MMAs over both (cta_group::2: each SM multiplies its
// rows by all columns), and each folds its own rows: half the bytes of B from L2 and in shared memory.
template <int BN, bool BROWS>
__global__ void __launch_bounds__(kThreads, 1) gemm_kernel(const __grid_constant__ GemmArgs p,
                                                           int dtype) {
  constexpr bool PAIR = BN == 256;
  constexpr int kSlots = kTmemCols / BN;
  constexpr int kBRows = PAIR ? BN / 2 : BN;  // rows of B this CTA loads
  constexpr uint32_t kStage = (kBM + kBRows) * kBlk;
  uint32_t rank = 0;
  if (PAIR) asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const int first = PAIR ? blockIdx.x >> 1 : blockIdx.x, step = PAIR ? gridDim.x >> 1 : gridDim.x;
  constexpr int kStages = kPipeBytes / kStage;
  constexpr int CW = BN / 2;  // columns per epilogue warp
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages], tfull[4], tempty[4], last;
  __shared__ uint32_t tmem_base;
  // a k-block's scales: the rows', and the weight blocks' or the columns'
  __shared__ __align__(16) float ring_s[kRing][kBM + (BROWS ? BN : 4)];
  __shared__ __align__(8) uint64_t sfull[kRing], sempty[kRing];
  uint8_t* stage = smem + kStages * kStage;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      tc::mbar_init(&full[i], 1);
      tc::mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < kSlots; ++i) {
      tc::mbar_init(&tfull[i], 1);
      tc::mbar_init(&tempty[i], (PAIR ? 2 : 1) * kEpiWarps);
    }
    for (int i = 0; i < kRing; ++i) {
      tc::mbar_init(&sfull[i], 32);
      tc::mbar_init(&sempty[i], kEpiWarps);
    }
    tc::mbar_init(&last, 1);
    tc::fence_barrier_init();
  }
  if (warp == 1) tmem_alloc<PAIR>(&tmem_base, kTmemCols);
  tc::fence_before_sync();
  __syncthreads();
  if (PAIR) cluster_sync();
  tc::fence_after_sync();
  const uint32_t tmem = tmem_base;
  const int tiles = p.mt * p.nt;
  grid_wait();   // what comes before reads nothing that the quantization writes

  if (warp < 4) {
    if (BN == 256) regs_dec<72>();
    if (warp == 0) {
      const bool one = elect_one();
      Turn<kStages> at;
      uint32_t issued = 0;
      bool ok = true;
      for (int t = first; ok && t < tiles; t += step) {
        int m, n;
        tile_at(p, t, m, n);
        for (int k = 0; k < p.kb; ++k) {
          const uint32_t s = at.i;
          // (a fresh barrier passes for the phase before its first)
          if (!warp_wait(&empty[s], at.phase ^ 1, p.err, 1)) {
            ok = false;
            break;
          }
          if (one) {
            uint8_t* st = smem + s * kStage;
            if (!PAIR || rank == 0)
              tc::mbar_arrive_expect_tx(&full[s], (PAIR ? 2 : 1) * kStage);
            if (PAIR) {
              const uint32_t bar = leader_u32(&full[s]);
              tma_load_2d_pair(st, &p.a, bar, k * kBlk, (2 * m + rank) * kBM);
              tma_load_2d_pair(st + kBM * kBlk, &p.b, bar, k * kBlk, n * BN + rank * kBRows);
            } else {
              tc::tma_load_2d(st, &p.a, &full[s], k * kBlk, m * kBM);
              tc::tma_load_2d(st + kBM * kBlk, &p.b, &full[s], k * kBlk, n * BN);
            }
          }
          __syncwarp();
          at.next();
          ++issued;
        }
      }
      // a copy still in flight after a timeout must land before the CTA's memory goes (a pair's
      // second CTA cannot see its own land: it waits far longer than a copy takes)
      if (!ok && one) {
        if (PAIR) {
          const long long t0 = clock64();
          while (clock64() - t0 < 20000000ll) {}
        } else {
          for (uint32_t i = issued > kStages ? issued - kStages : 0; i < issued; ++i)
            tc::mbar_wait(&full[i % kStages], (i / kStages) & 1, nullptr, 0);
        }
      }
    } else if (warp == 1 && rank == 0) {
      // The tensor core takes 256 or 512 cycles for a k-block: the loop that feeds it has to be
      // shorter, so its control and operands are uniform over the warp and one lane issues.
      constexpr uint32_t id = idesc_e4m3(PAIR ? 2 * kBM : kBM, BN);
      const bool one = elect_one();
      const uint32_t base = tc::smem_u32(smem);
      const uint64_t da0 = tc::umma_desc_k_sw128(base),
                     db0 = tc::umma_desc_k_sw128(base + kBM * kBlk);
      Turn<kStages> at;
      Turn<kSlots> acc;
      bool ok = true;
      for (int t = first; ok && t < tiles; t += step) {
        for (int k = 0; k < p.kb; ++k) {
          if (!warp_wait(&tempty[acc.i], acc.phase ^ 1, p.err, 2) ||
              !warp_wait(&full[at.i], at.phase, p.err, 3)) {
            ok = false;
            break;
          }
          tc::fence_after_sync();
          const uint64_t off = at.i * (kStage >> 4);
          const uint32_t d = tmem + acc.i * BN;
          if (one) {
#pragma unroll
            for (int j = 0; j < 4; ++j)  // 32 values (32 bytes) of k per instruction
              umma_e4m3<PAIR>(d, da0 + off + 2 * j, db0 + off + 2 * j, id, j > 0);
            umma_commit<PAIR>(&empty[at.i]);
            umma_commit<PAIR>(&tfull[acc.i]);
          }
          __syncwarp();
          at.next();
          acc.next();
        }
      }
      if (one) {
        umma_commit<PAIR>(&last);
        tc::mbar_wait(&last, 0, p.err, 4);
      }
    } else if (warp == 2) {
      // Scales: copied to the ring up to kRing k-blocks ahead of the fold (a load from L2 takes
      // longer than the MMAs of a k-block); each lane's arrival on sfull follows its copies.
      Turn<kRing> at;
      bool ok = true;
      for (int t = first; ok && t < tiles; t += step) {
        int mi, ni;
        tile_at(p, t, mi, ni);
        const int m = (PAIR ? 2 * mi + rank : mi) * kBM + lane;
        const float* sa = p.sa + m;
        const float* sb = p.sb;
        int n = ni * BN;
        if (BROWS) {
          n += lane;
          sb += n;
        } else {   // lane i: the weight block of columns 128 i .. of the tile
          n += kBlk * lane;
          sb += n / kBlk * p.sb_n;
        }
        for (int k = 0; k < p.kb; ++k, at.next()) {
          const uint32_t e = at.i;
          ok = warp_wait(&sempty[e], at.phase ^ 1, p.err, 8);
          if (!ok) break;
          float* to = ring_s[e];
#pragma unroll
          for (int i = 0; i < 4; ++i) copy4(to + 32 * i + lane, sa + 32 * i, m + 32 * i < p.M);
          if (BROWS) {
#pragma unroll
            for (int i = 0; i < BN / 32; ++i)
              copy4(to + kBM + 32 * i + lane, sb + 32 * i, n + 32 * i < p.N);
          } else if (lane < BN / kBlk) {
            copy4(to + kBM + lane, sb, n < p.N);
          }
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(
                           tc::smem_u32(&sfull[e]))
                       : "memory");
          sa += p.ld_sa;
          sb += p.sb_k;
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
    }
  } else {
    if (BN == 256) regs_inc<216>();
    const int q = warp & 3, part = (warp - 4) >> 2;
    const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16) + part * CW;
    Turn<kSlots> slot;
    Turn<kRing> at;
    int buf = 0;
    bool ok = true;
    for (int t = first; ok && t < tiles; t += step) {
      int mi, ni;
      tile_at(p, t, mi, ni);
      const int m = (PAIR ? 2 * mi + rank : mi) * kBM + q * 32 + lane, n0 = ni * BN + part * CW;
      uint64_t acc[CW / 2];   // pairs of float32, in registers as the packed operations take them
#pragma unroll
      for (int c = 0; c < CW / 2; ++c) acc[c] = 0;
      for (int k = 0; k < p.kb; ++k) {
        const uint32_t sl = slot.i, e = at.i;
        ok = warp_wait(&sfull[e], at.phase, p.err, 7) &&
             warp_wait(&tfull[sl], slot.phase, p.err, 5);
        if (!ok) break;
        tc::fence_after_sync();
        slot.next();
        at.next();
        float s = ring_s[e][q * 32 + lane];
        if (!BROWS) s *= ring_s[e][kBM + part * CW / kBlk];
        const uint64_t s2 = f2_same(s).b;
        const float* sbw = ring_s[e] + kBM + part * CW;
        uint32_t r[64];
#pragma unroll
        for (int c = 0; c < CW / 64; ++c) {
          tmem_ld64(lanes + sl * BN + 64 * c, r);
          tc::tmem_wait_ld();
          if (c + 1 == CW / 64) {
            // the accumulator is given back before its last columns are folded
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) {
              if (PAIR) arrive_leader(&tempty[sl]);
              else mbar_arrive(&tempty[sl]);
            }
          }
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            if (BROWS)
              fold2(acc[32 * c + j], r[2 * j], r[2 * j + 1],
                    *reinterpret_cast<const uint64_t*>(sbw + (BROWS ? 64 * c + 2 * j : 0)), s2);
            else
              fold(acc[32 * c + j], r[2 * j], r[2 * j + 1], s2);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sempty[e]);
      }
      if (ok) {
        uint8_t* st = stage + (warp - 4) * 2 * 4096;
        const int m0 = m - lane;
        if (p.boxes) {
          if (dtype == BF16) store_boxes<__nv_bfloat16, CW>(p, st, buf, lane, m0, n0, acc);
          else if (dtype == F16) store_boxes<__half, CW>(p, st, buf, lane, m0, n0, acc);
          else store_boxes<float, CW>(p, st, buf, lane, m0, n0, acc);
        } else {
          if (dtype == BF16) store_row<__nv_bfloat16, CW>(p, m, n0, acc);
          else if (dtype == F16) store_row<__half, CW>(p, m, n0, acc);
          else store_row<float, CW>(p, m, n0, acc);
        }
      }
    }
    if (lane == 0) tc::bulk_wait_all();
  }
  tc::fence_before_sync();
  __syncthreads();
  if (PAIR) {
    // the second CTA stays until the pair's last commit has arrived here too
    if (rank == 1 && threadIdx.x == 0) tc::mbar_wait(&last, 0, p.err, 9);
    cluster_sync();   // (the other CTA's MMAs, commits and arrivals are over)
  }
  tc::fence_after_sync();
  if (warp == 1) tmem_dealloc<PAIR>(tmem, kTmemCols);
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                  const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  if (!fn) {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = (EncodeTiledFn)f;
  }
  return fn;
}

// codes [rows][ld], `cols` of them valid: boxes of box_rows x 128 bytes, 128-byte swizzle; rows
// and columns outside read as zero.
static bool codes_map(CUtensorMap* m, const void* base, int64_t rows, int cols, int64_t ld,
                      int box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld};
  cuuint32_t box[2] = {(cuuint32_t)kBlk, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// out [M][ld] in boxes of 32 rows x 128 bytes.
static bool out_map(CUtensorMap* m, void* base, int dtype, int M, int N, int64_t ld) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t es = dtype_size(dtype);
  cuuint64_t dims[2] = {(cuuint64_t)N, (cuuint64_t)M};
  cuuint64_t strides[1] = {(cuuint64_t)ld * es};
  cuuint32_t box[2] = {(cuuint32_t)(128 / es), 32};
  cuuint32_t estr[2] = {1, 1};
  const CUtensorMapDataType t = dtype == BF16  ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                : dtype == F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                               : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
  return fn(m, t, 2, base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// A launch in clusters of `cluster` CTAs; follows: it may begin while the kernel before it on the
// stream, whose output it reads only after grid_wait, still runs.
template <typename K, typename... A>
static int launch_cluster(K kern, int blocks, int threads, uint32_t smem, int cluster, bool follows,
                          cudaStream_t st, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (cluster > 1) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = cluster;
    at[n].val.clusterDim.y = at[n].val.clusterDim.z = 1;
    ++n;
  }
  if (follows) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = at;
  cfg.numAttrs = n;
  if (cudaLaunchKernelEx(&cfg, kern, args...) != cudaSuccess) return GSQ_ECUDA;
  GSQ_CHECK_LAUNCH();
  return GSQ_OK;
}

// Whether the wide kernel was compiled to the register count that its split was made for (another
// count would leave a setmaxnreg waiting, or registers unused): if not, the narrow tiles serve.
template <bool BROWS>
static int wide_fits(bool& fits) {
  cudaFuncAttributes at;
  if (cudaFuncGetAttributes(&at, gemm_kernel<256, BROWS>) != cudaSuccess) return GSQ_ECUDA;
  fits = at.numRegs == kLaunchRegs;
  return GSQ_OK;
}

template <int BN, bool BROWS>
static int launch_gemm(GemmArgs& p, const void* b, int64_t ldb, int dtype, bool follows,
                       cudaStream_t st) {
  constexpr bool PAIR = BN == 256;
  constexpr int kBRows = PAIR ? BN / 2 : BN;
  constexpr uint32_t kStage = (kBM + kBRows) * kBlk;
  constexpr uint32_t smem = kPipeBytes / kStage * kStage + kStageBytes + 1024;
  auto kern = gemm_kernel<BN, BROWS>;
  if (!codes_map(&p.b, b, p.N, p.K, ldb, kBRows)) return GSQ_ECUDA;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) !=
      cudaSuccess)
    return GSQ_ECUDA;
  constexpr int rows = PAIR ? 2 * kBM : kBM;
  p.mt = (p.M + rows - 1) / rows;
  p.nt = (p.N + BN - 1) / BN;
  p.group = 16 / (PAIR ? 2 : 1);
  const int64_t tiles = (int64_t)p.mt * p.nt;
  if (tiles > INT32_MAX / 2) return GSQ_EINVAL;
  const int most = num_sms() / (PAIR ? 2 : 1);
  const int n = (int)(tiles < most ? tiles : most);
  return launch_cluster(kern, PAIR ? 2 * n : n, kThreads, smem, PAIR ? 2 : 1, follows, st, p, dtype);
}

// ------------------------------------------------------------------------ few rows (decode) ---
// Up to 64 rows of A: the weight's bytes bound the product, so its rows are the 128 of an MMA
// tile and the activations its NT columns, and the k-blocks of a row tile are shared out over a
// cluster of CTAs (a 8192 x 8192 weight has 64 row tiles for 148 SMs). Each CTA streams its
// k-blocks through kSkStages stages and folds each with the scales of its 128 x 128 block and of
// the columns; the partial sums meet in the first CTAs' shared memory in the order of the ranks.
// The weight's first stages are loaded before the activations are quantized (grid_wait).
// 16 x 8192 x 8192: 67 MB in 16.5 us, 4.1 TB/s; 1 x 896 x 1152: 5.3 us with the quantization.
constexpr int kSkStages = 5;
constexpr int kSkThreads = 256;

struct SkinnyArgs {
  CUtensorMap w, x;
  int M, N, kb, splits;
  const float* sx;
  int64_t ld_sx;
  const float* sw;
  int64_t sw_n, sw_k;
  void* out;
  int64_t ld_o;
  int* err;
};

template <int NT>
__global__ void __launch_bounds__(kSkThreads) skinny_kernel(const __grid_constant__ SkinnyArgs p,
                                                            int dtype) {
  constexpr int kSlots = 4;
  constexpr uint32_t kCols = kSlots * NT < 32 ? 32 : kSlots * NT;
  constexpr uint32_t kW = kBM * kBlk, kStage = kW + NT * kBlk;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(8) uint64_t full[kSkStages], empty[kSkStages], tfull[kSlots], tempty[kSlots];
  __shared__ __align__(8) uint64_t last;
  __shared__ uint32_t tmem_base;
  __shared__ __align__(16) float part[NT][kBM];   // this CTA's sums
  __shared__ __align__(16) float sx_s[16][NT];    // scales of 16 k-blocks, of their columns
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x % p.splits, tile = blockIdx.x / p.splits;
  const int k0 = (int)((int64_t)p.kb * rank / p.splits),
            k1 = (int)((int64_t)p.kb * (rank + 1) / p.splits);
  if (threadIdx.x == 0) {
    for (int i = 0; i < kSkStages; ++i) {
      tc::mbar_init(&full[i], 1);
      tc::mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < kSlots; ++i) {
      tc::mbar_init(&tfull[i], 1);
      tc::mbar_init(&tempty[i], 4);
    }
    tc::mbar_init(&last, 1);
    tc::fence_barrier_init();
  }
  if (warp == 1) tc::tmem_alloc(&tmem_base, kCols);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = tmem_base;
  if (warp == 0) {
    const bool one = elect_one();
    const int first = min(k1 - k0, kSkStages);
    if (one)
      for (int i = 0; i < first; ++i) {
        tc::mbar_arrive_expect_tx(&full[i], kStage);
        tc::tma_load_2d(smem + i * kStage, &p.w, &full[i], (k0 + i) * kBlk, tile * kBM);
      }
    grid_wait();
    if (one)
      for (int i = 0; i < first; ++i)
        tc::tma_load_2d(smem + i * kStage + kW, &p.x, &full[i], (k0 + i) * kBlk, 0);
    __syncwarp();
    Turn<kSkStages> at;
    bool ok = true;
    int issued = first;
    for (int k = k0 + first; k < k1; ++k, at.next()) {
      if (!warp_wait(&empty[at.i], at.phase, p.err, 11)) {
        ok = false;
        break;
      }
      if (one) {
        uint8_t* st = smem + at.i * kStage;
        tc::mbar_arrive_expect_tx(&full[at.i], kStage);
        tc::tma_load_2d(st, &p.w, &full[at.i], k * kBlk, tile * kBM);
        tc::tma_load_2d(st + kW, &p.x, &full[at.i], k * kBlk, 0);
      }
      __syncwarp();
      ++issued;
    }
    // a copy still in flight after a timeout must land before the CTA's memory goes
    if (!ok && one)
      for (int i = issued > kSkStages ? issued - kSkStages : 0; i < issued; ++i)
        tc::mbar_wait(&full[i % kSkStages], (i / kSkStages) & 1, nullptr, 0);
  } else if (warp == 1) {
    constexpr uint32_t id = idesc_e4m3(kBM, NT);
    const bool one = elect_one();
    const uint32_t base = tc::smem_u32(smem);
    const uint64_t da0 = tc::umma_desc_k_sw128(base), db0 = tc::umma_desc_k_sw128(base + kW);
    Turn<kSkStages> at;
    Turn<kSlots> acc;
    for (int k = k0; k < k1; ++k, at.next(), acc.next()) {
      if (!warp_wait(&tempty[acc.i], acc.phase ^ 1, p.err, 12) ||
          !warp_wait(&full[at.i], at.phase, p.err, 13))
        break;
      tc::fence_after_sync();
      if (one) {
        const uint64_t off = at.i * (kStage >> 4);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          umma_e4m3<false>(tmem + acc.i * NT, da0 + off + 2 * j, db0 + off + 2 * j, id, j > 0);
        tc::umma_commit(&empty[at.i]);
        tc::umma_commit(&tfull[acc.i]);
      }
      __syncwarp();
    }
    if (one) {
      tc::umma_commit(&last);
      tc::mbar_wait(&last, 0, p.err, 14);
    }
  } else if (warp >= 4) {
    grid_wait();
    const int q = warp & 3, row = q * 32 + lane, tid = threadIdx.x - 128;
    const float* sw = p.sw + min(tile * kBM, p.N - 1) / kBlk * p.sw_n;
    float acc[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[j] = 0.f;
    Turn<kSlots> slot;
    bool ok = true;
    for (int kc = k0; kc < k1; kc += 16) {
      // the scales of up to 16 k-blocks, times the weight block's
      asm volatile("bar.sync 1, 128;" ::: "memory");
      for (int i = tid; i < 16 * NT; i += 128) {
        const int k = kc + i / NT, m = i % NT;
        sx_s[i / NT][m] = k < k1 && m < p.M ? p.sx[k * p.ld_sx + m] * sw[k * p.sw_k] : 0.f;
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");
      for (int k = kc; k < min(k1, kc + 16); ++k) {
        // (after a timeout the loop runs on, unread: the four warps' barriers keep their count)
        if (ok) ok = warp_wait(&tfull[slot.i], slot.phase, p.err, 15);
        if (!ok) continue;
        tc::fence_after_sync();
        const float* sx = sx_s[k - kc];
#pragma unroll
        for (int c = 0; c < NT; c += 16) {
          float v[16];
          tc::tmem_ld16(tmem + ((uint32_t)(q * 32) << 16) + slot.i * NT + c, v);
#pragma unroll
          for (int j = 0; j < 16; ++j) acc[c + j] = fmaf(v[j], sx[c + j], acc[c + j]);
        }
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&tempty[slot.i]);
        slot.next();
      }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) part[j][row] = acc[j];
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  if (warp == 1) tc::tmem_dealloc(tmem, kCols);
  if (p.splits > 1) cluster_sync();
  // rows of the output (tokens) rank, rank + splits, ...: 128 columns each, summed over the ranks
  const int n = threadIdx.x & 127, col = tile * kBM + n;
  for (int m = rank + p.splits * (threadIdx.x >> 7); m < p.M; m += 2 * p.splits) {
    float v = 0.f;
    for (int r = 0; r < p.splits; ++r) {
      float x;
      uint32_t a;
      asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(tc::smem_u32(&part[m][n])), "r"(r));
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(a) : "memory");
      v += x;
    }
    if (col < p.N) {
      const int64_t o = m * p.ld_o + col;
      if (dtype == BF16) reinterpret_cast<__nv_bfloat16*>(p.out)[o] = from_f32<__nv_bfloat16>(v);
      else if (dtype == F16) reinterpret_cast<__half*>(p.out)[o] = from_f32<__half>(v);
      else reinterpret_cast<float*>(p.out)[o] = v;
    }
  }
  if (p.splits > 1) cluster_sync();   // (the other CTAs have read this one's sums)
}

constexpr int kSkRows = 64;

template <int NT>
static int launch_skinny(const GemmArgs& g, const void* x, int64_t ld_x, const void* w, int64_t ldw,
                         int dtype, bool follows, cudaStream_t st) {
  constexpr uint32_t kStage = (kBM + NT) * kBlk, smem = kSkStages * kStage + 1024;
  SkinnyArgs p;
  if (!codes_map(&p.w, w, g.N, g.K, ldw, kBM) || !codes_map(&p.x, x, g.M, g.K, ld_x, NT))
    return GSQ_ECUDA;
  auto kern = skinny_kernel<NT>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) !=
      cudaSuccess)
    return GSQ_ECUDA;
  p.M = g.M;
  p.N = g.N;
  p.kb = g.kb;
  p.sx = g.sa;
  p.ld_sx = g.ld_sa;
  p.sw = g.sb;
  p.sw_n = g.sb_n;
  p.sw_k = g.sb_k;
  p.out = g.out;
  p.ld_o = g.ld_o;
  p.err = g.err;
  const int tiles = (g.N + kBM - 1) / kBM;
  // as many parts of k as give every SM a CTA, and no more than there are k-blocks
  int s = 1;
  while (s < 8 && tiles * s < num_sms() && 2 * s <= g.kb) s *= 2;
  p.splits = s;
  return launch_cluster(kern, tiles * s, kSkThreads, smem, s, follows, st, p, dtype);
}

// A product's tile: rows x columns of the output that one CTA, or a pair of CTAs, works on; for few
// rows, all of them by 128 columns.
enum Tile { FEW_16, FEW_32, FEW_64, PAIR_256, ONE_128 };

static Tile tile_of(int M, int N, bool sb_rows, bool accumulate, int sms, bool wide) {
  // Few rows: bound by the weight's bytes (16 x 8192 x 8192 with its quantization: 31 us on
  // 128-row tiles of A, which leave half of the SMs idle, 16.5 us with the weight's rows as the tile
  // and k shared out over clusters).
  if (M <= kSkRows && !sb_rows && !accumulate)
    return M <= 16 ? FEW_16 : M <= 32 ? FEW_32 : FEW_64;
  // Tile by the time of the rounds that the busiest SM walks: 256 x 256 of a pair, or 128 x 128 of
  // one SM, whose k-block takes 0.66 to 0.7 of the wide one's time (8191 x 4096 -> 8192: 28 rounds
  // in 348 us for 14 in 253; 16384 x 896 -> 4864: 33 in 114 for 17 in 89; 1024 x 4096 -> 4096: 2 in
  // 30 for 1 in 22.5), with a scale per row of both sides 0.5 to 0.55 (28 in 454 for 14 in 424; 33
  // in 156 for 17 in 160; 2 in 37 for 1 in 34). So it is taken where it needs few more rounds (1408
  // x 2048 -> 3200: 2 in 17.8 for 2 in 22.8; 600 x 4096 -> 9000 with a scale per row: 3 in 54 for 2
  // in 65, without: 43 for 40). 256 x 128 of a pair was never faster than 128 x 128 (forty
  // products: equal to 40 % slower) and is not built.
  const auto rounds = [&](int rows, int bn, int per) {
    return (double)(((int64_t)((M + rows - 1) / rows) * ((N + bn - 1) / bn) * per + sms - 1) / sms);
  };
  return wide && rounds(256, 256, 2) <= (sb_rows ? 0.55 : 0.7) * rounds(128, 128, 1) ? PAIR_256
                                                                                     : ONE_128;
}

template <typename T>
static int quant_launch(const T* x, int rows, int cols, int64_t ld_x, uint8_t* codes, int64_t ld_c,
                        float* scales, int64_t ld_s, uint8_t* codes_t, int64_t ld_ct,
                        float* scales_t, int64_t ld_st, bool blocks, cudaStream_t st) {
  const bool vec = (uintptr_t)x % 16 == 0 && ld_x * sizeof(T) % 16 == 0 && cols % 4 == 0;
  const int cb = (cols + kBlk - 1) / kBlk, rb = (rows + kBlk - 1) / kBlk;
  if (!blocks && !codes_t) {
    const int64_t items = (int64_t)((rows + kRowsWarp - 1) / kRowsWarp) * cb;
    int64_t g = (items + 7) / 8;
    const int64_t cap = (int64_t)num_sms() * 32;
    if (g > cap) g = cap;
    if (vec) quant_rows_kernel<T, true><<<(unsigned)g, 256, 0, st>>>(x, ld_x, rows, cols, cb, codes, ld_c, scales, ld_s);
    else quant_rows_kernel<T, false><<<(unsigned)g, 256, 0, st>>>(x, ld_x, rows, cols, cb, codes, ld_c, scales, ld_s);
    GSQ_CHECK_LAUNCH();
    return GSQ_OK;
  }
  const dim3 g(cb, rb);
#define GSQ_QT(R, C, B)                                                                          \
  do {                                                                                           \
    if (vec) quant_tile_kernel<T, true, R, C, B><<<g, 256, 0, st>>>(                             \
        x, ld_x, rows, cols, codes, ld_c, scales, ld_s, codes_t, ld_ct, scales_t, ld_st);        \
    else quant_tile_kernel<T, false, R, C, B><<<g, 256, 0, st>>>(                                \
        x, ld_x, rows, cols, codes, ld_c, scales, ld_s, codes_t, ld_ct, scales_t, ld_st);        \
  } while (0)
  if (blocks) GSQ_QT(false, false, true);
  else if (codes) GSQ_QT(true, true, false);
  else GSQ_QT(false, true, false);
#undef GSQ_QT
  GSQ_CHECK_LAUNCH();
  return GSQ_OK;
}

static int quant_any(const void* x, int dtype, int rows, int cols, int64_t ld_x, void* codes,
                     int64_t ld_c, float* scales, int64_t ld_s, void* codes_t, int64_t ld_ct,
                     float* scales_t, int64_t ld_st, bool blocks, cudaStream_t st) {
  auto* c = (uint8_t*)codes;
  auto* ct = (uint8_t*)codes_t;
  if (dtype == BF16)
    return quant_launch((const __nv_bfloat16*)x, rows, cols, ld_x, c, ld_c, scales, ld_s, ct,
                        ld_ct, scales_t, ld_st, blocks, st);
  if (dtype == F16)
    return quant_launch((const __half*)x, rows, cols, ld_x, c, ld_c, scales, ld_s, ct, ld_ct,
                        scales_t, ld_st, blocks, st);
  return quant_launch((const float*)x, rows, cols, ld_x, c, ld_c, scales, ld_s, ct, ld_ct,
                      scales_t, ld_st, blocks, st);
}

// a code matrix that TMA and the 8-byte stores can take
inline bool codes_ok(const void* c, int64_t ld, int cols) {
  return c && (uintptr_t)c % 16 == 0 && ld % 16 == 0 && ld >= cols;
}

inline bool gemm_ok(int M, int N, int K, const void* a, int64_t lda, const float* sa,
                    int64_t ld_sa, const void* b, int64_t ldb, const float* sb, int sb_rows,
                    int64_t sb_n, int64_t sb_k, const void* out, int dtype, int64_t ld_out,
                    int accumulate, const int* err) {
  return M > 0 && N > 0 && K > 0 && M <= kMaxDim && N <= kMaxDim && K <= kMaxDim &&
         codes_ok(a, lda, K) && codes_ok(b, ldb, K) && sa &&
         ld_sa >= M && sb && sb_n >= 0 && sb_k >= 0 && out && dtype >= 0 && dtype <= 2 &&
         ld_out >= N && err && lies_on(out, dtype_size(dtype)) && lies_on(sa, 4) &&
         lies_on(sb, 4) && lies_on(err, 4) &&
         !(accumulate && dtype != F32) && !(sb_rows && sb_k < N);
}

inline bool quant_ok(const void* x, int dtype, int rows, int cols, int64_t ld_x) {
  return x && dtype >= 0 && dtype <= 2 && rows > 0 && cols > 0 && rows <= kMaxDim &&
         cols <= kMaxDim && ld_x >= cols &&
         (uintptr_t)x % dtype_size(dtype) == 0;
}

}  // namespace fp8
}  // namespace gsq

using namespace gsq;

extern "C" int gsq_fp8_quant(const void* x, int dtype, int rows, int cols, int64_t ld_x,
                             void* codes, int64_t ld_codes, float* scales, int64_t ld_scales,
                             void* codes_t, int64_t ld_codes_t, float* scales_t,
                             int64_t ld_scales_t, void* stream) {
  if (!fp8::quant_ok(x, dtype, rows, cols, ld_x) || (!codes && !codes_t)) return GSQ_EINVAL;
  if (codes && (!fp8::codes_ok(codes, ld_codes, cols) || !scales || ld_scales < rows))
    return GSQ_EINVAL;
  if (codes_t && (!fp8::codes_ok(codes_t, ld_codes_t, rows) || !scales_t || ld_scales_t < cols))
    return GSQ_EINVAL;
  if (!lies_on(scales, 4) || !lies_on(scales_t, 4)) return GSQ_EINVAL;
  if (codes_t && (rows + 127) / 128 > 65535) return GSQ_EINVAL;
  return fp8::quant_any(x, dtype, rows, cols, ld_x, codes, ld_codes, scales, ld_scales, codes_t,
                        ld_codes_t, scales_t, ld_scales_t, false, (cudaStream_t)stream);
}

extern "C" int gsq_fp8_quant_blocks(const void* w, int dtype, int N, int K, int64_t ld_w,
                                    void* codes, int64_t ld_codes, float* scales,
                                    int64_t ld_scales, void* stream) {
  if (!fp8::quant_ok(w, dtype, N, K, ld_w) || !fp8::codes_ok(codes, ld_codes, K) || !scales ||
      !lies_on(scales, 4) ||
      ld_scales < (K + 127) / 128 || (N + 127) / 128 > 65535)
    return GSQ_EINVAL;
  return fp8::quant_any(w, dtype, N, K, ld_w, codes, ld_codes, scales, ld_scales, nullptr, 0,
                        nullptr, 0, true, (cudaStream_t)stream);
}

extern "C" int gsq_fp8_dequant(const void* codes, int64_t ld_codes, const float* scales,
                               int64_t ld_scales, int N, int K, void* out, int dtype,
                               int64_t ld_out, void* stream) {
  if (!fp8::codes_ok(codes, ld_codes, K) || !scales || !lies_on(scales, 4) || N <= 0 || K <= 0 ||
      N > kMaxDim || K > kMaxDim ||
      ld_scales < (K + 127) / 128 || !out || dtype < 0 || dtype > 2 || ld_out < K ||
      (uintptr_t)out % dtype_size(dtype))
    return GSQ_EINVAL;
  int64_t g = ((int64_t)N * ((K + 7) / 8) + 255) / 256;
  const int64_t cap = (int64_t)num_sms() * 16;
  if (g > cap) g = cap;
  cudaStream_t st = (cudaStream_t)stream;
  const auto* c = (const uint8_t*)codes;
  if (dtype == BF16)
    fp8::dequant_blocks_kernel<<<(unsigned)g, 256, 0, st>>>(c, ld_codes, scales, ld_scales, N, K,
                                                            (__nv_bfloat16*)out, ld_out);
  else if (dtype == F16)
    fp8::dequant_blocks_kernel<<<(unsigned)g, 256, 0, st>>>(c, ld_codes, scales, ld_scales, N, K,
                                                            (__half*)out, ld_out);
  else
    fp8::dequant_blocks_kernel<<<(unsigned)g, 256, 0, st>>>(c, ld_codes, scales, ld_scales, N, K,
                                                            (float*)out, ld_out);
  GSQ_CHECK_LAUNCH();
  return GSQ_OK;
}

static int fp8_gemm(int M, int N, int K, const void* a, int64_t lda, const float* sa,
                    int64_t ld_sa, const void* b, int64_t ldb, const float* sb,
                    int sb_rows, int64_t sb_n, int64_t sb_k, void* out,
                    int dtype, int64_t ld_out, int accumulate, int* err, bool follows,
                    void* stream) {
  if (!fp8::gemm_ok(M, N, K, a, lda, sa, ld_sa, b, ldb, sb, sb_rows, sb_n, sb_k, out, dtype, ld_out,
                    accumulate, err))
    return GSQ_EINVAL;
  fp8::GemmArgs p;
  if (!fp8::codes_map(&p.a, a, M, K, lda, fp8::kBM)) return GSQ_ECUDA;
  p.M = M;
  p.N = N;
  p.K = K;
  p.kb = (K + fp8::kBlk - 1) / fp8::kBlk;
  p.sa = sa;
  p.ld_sa = ld_sa;
  p.sb = sb;
  p.sb_n = sb_n;
  p.sb_k = sb_k;
  p.out = out;
  p.ld_o = ld_out;
  p.accumulate = accumulate;
  p.boxes = !accumulate && (uintptr_t)out % 16 == 0 && ld_out * dtype_size(dtype) % 16 == 0;
  if (p.boxes && !fp8::out_map(&p.o, out, dtype, M, N, ld_out)) return GSQ_ECUDA;
  p.err = err;
  cudaStream_t st = (cudaStream_t)stream;
  fp8::Tile t = fp8::tile_of(M, N, sb_rows, accumulate, num_sms(), true);
  if (t == fp8::PAIR_256) {
    bool fits;
    const int r = sb_rows ? fp8::wide_fits<true>(fits) : fp8::wide_fits<false>(fits);
    if (r != GSQ_OK) return r;
    if (!fits) t = fp8::tile_of(M, N, sb_rows, accumulate, num_sms(), false);
  }
  switch (t) {
    case fp8::FEW_16: return fp8::launch_skinny<16>(p, a, lda, b, ldb, dtype, follows, st);
    case fp8::FEW_32: return fp8::launch_skinny<32>(p, a, lda, b, ldb, dtype, follows, st);
    case fp8::FEW_64: return fp8::launch_skinny<64>(p, a, lda, b, ldb, dtype, follows, st);
    case fp8::PAIR_256:
      return sb_rows ? fp8::launch_gemm<256, true>(p, b, ldb, dtype, follows, st)
                     : fp8::launch_gemm<256, false>(p, b, ldb, dtype, follows, st);
    default:
      return sb_rows ? fp8::launch_gemm<128, true>(p, b, ldb, dtype, follows, st)
                     : fp8::launch_gemm<128, false>(p, b, ldb, dtype, follows, st);
  }
}

extern "C" int gsq_fp8_gemm_tile(int M, int N, int sb_rows, int accumulate, int sms, int wide,
                                 int* rows, int* cols) {
  if (M <= 0 || N <= 0 || M > kMaxDim || N > kMaxDim || sms <= 0 || !rows || !cols)
    return GSQ_EINVAL;
  const fp8::Tile t = fp8::tile_of(M, N, sb_rows, accumulate, sms, wide);
  *rows = t == fp8::FEW_16 ? 16 : t == fp8::FEW_32 ? 32 : t == fp8::FEW_64 ? 64
          : t == fp8::PAIR_256 ? 256 : 128;
  *cols = t == fp8::PAIR_256 ? 256 : 128;
  return GSQ_OK;
}

extern "C" int gsq_fp8_gemm(int M, int N, int K, const void* a, int64_t lda, const float* sa,
                            int64_t ld_sa, const void* b, int64_t ldb, const float* sb,
                            int sb_rows, int64_t sb_n, int64_t sb_k, void* out, int dtype,
                            int64_t ld_out, int accumulate, int* err, void* stream) {
  return fp8_gemm(M, N, K, a, lda, sa, ld_sa, b, ldb, sb, sb_rows, sb_n, sb_k, out, dtype, ld_out,
                  accumulate, err, false, stream);
}

extern "C" int gsq_fp8_linear(const void* x, int dtype, int M, int K, int64_t ld_x,
                              const void* codes, int64_t ld_codes, const float* scales,
                              int64_t ld_scales, int N, void* y, int y_dtype, int64_t ld_y,
                              void* workspace, int64_t workspace_bytes, int* err, void* stream) {
  if (M <= 0 || K <= 0 || N <= 0 || M > kMaxDim || K > kMaxDim || N > kMaxDim || !workspace ||
      (uintptr_t)workspace % 16)
    return GSQ_EINVAL;
  const int64_t ld_q = ((int64_t)K + 15) / 16 * 16;
  const int64_t need = M * ld_q + (int64_t)4 * M * ((K + fp8::kBlk - 1) / fp8::kBlk);
  if (workspace_bytes < need || ld_scales < (K + fp8::kBlk - 1) / fp8::kBlk) return GSQ_EINVAL;
  auto* q = (uint8_t*)workspace;
  auto* sq = (float*)(q + M * ld_q);
  if (!fp8::quant_ok(x, dtype, M, K, ld_x) ||
      !fp8::gemm_ok(M, N, K, q, ld_q, sq, M, codes, ld_codes, scales, 0, ld_scales, 1, y, y_dtype,
                    ld_y, 0, err))
    return GSQ_EINVAL;
  const int s = gsq_fp8_quant(x, dtype, M, K, ld_x, q, ld_q, sq, M, nullptr, 0, nullptr, 0, stream);
  if (s != GSQ_OK) return s;
  return fp8_gemm(M, N, K, q, ld_q, sq, M, codes, ld_codes, scales, 0, ld_scales, 1, y, y_dtype,
                  ld_y, 0, err, true, stream);
}

extern "C" int gsq_fp8_linear_vjp(const void* x, int dtype, int M, int K, int64_t ld_x,
                                  const void* dy, int dy_dtype, int N, int64_t ld_dy,
                                  const void* codes_t, int64_t ld_codes_t, const float* scales,
                                  int64_t ld_scales, void* dx, int64_t ld_dx, float* dw,
                                  int64_t ld_dw, int accumulate, void* workspace,
                                  int64_t workspace_bytes, int* err, void* stream) {
  if (M <= 0 || K <= 0 || N <= 0 || M > kMaxDim || K > kMaxDim || N > kMaxDim || !workspace ||
      (uintptr_t)workspace % 16)
    return GSQ_EINVAL;
  const auto blocks = [](int64_t n) { return (n + fp8::kBlk - 1) / fp8::kBlk; };
  const int64_t ln = ((int64_t)N + 15) / 16 * 16, lm = ((int64_t)M + 15) / 16 * 16;
  const int64_t codes = M * ln + ((int64_t)N + K) * lm,
                need = codes + 4 * (blocks(N) * M + blocks(M) * ((int64_t)N + K));
  if (workspace_bytes < need || ld_scales < blocks(K) || blocks(M) > 65535) return GSQ_EINVAL;
  // dy in rows along N, dy and x in columns (blocks of 128 rows), transposed
  auto* dyq = (uint8_t*)workspace;
  auto* dyt = dyq + M * ln;
  auto* xt = dyt + N * lm;
  auto* s_dy = (float*)(dyq + codes);
  float *s_dyt = s_dy + blocks(N) * M, *s_xt = s_dyt + blocks(M) * N;
  if (!fp8::quant_ok(x, dtype, M, K, ld_x) || !fp8::quant_ok(dy, dy_dtype, M, N, ld_dy) ||
      !fp8::gemm_ok(M, K, N, dyq, ln, s_dy, M, codes_t, ld_codes_t, scales, 0, 1, ld_scales, dx,
                    dtype, ld_dx, 0, err) ||
      !fp8::gemm_ok(N, K, M, dyt, lm, s_dyt, N, xt, lm, s_xt, 1, 0, K, dw, F32, ld_dw, accumulate,
                    err))
    return GSQ_EINVAL;
  cudaStream_t st = (cudaStream_t)stream;
  int s = fp8::quant_any(dy, dy_dtype, M, N, ld_dy, dyq, ln, s_dy, M, dyt, lm, s_dyt, N, false, st);
  if (s == GSQ_OK)
    s = fp8::quant_any(x, dtype, M, K, ld_x, nullptr, 0, nullptr, 0, xt, lm, s_xt, K, false, st);
  if (s == GSQ_OK)
    s = fp8_gemm(M, K, N, dyq, ln, s_dy, M, codes_t, ld_codes_t, scales, 0, 1, ld_scales, dx, dtype,
                 ld_dx, 0, err, false, stream);
  if (s == GSQ_OK)
    s = fp8_gemm(N, K, M, dyt, lm, s_dyt, N, xt, lm, s_xt, 1, 0, K, dw, F32, ld_dw, accumulate, err,
                 false, stream);
  return s;
}
