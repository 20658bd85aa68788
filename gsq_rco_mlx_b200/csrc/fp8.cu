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
// registers with one multiply-add per value. At the tensor cores' e4m3 rate a 128 x 256 tile
// takes 512 cycles per k-block; the fold takes 128 x 256 / (4 x 32 lanes) = 256 issue slots of
// the same cycles on the four schedulers, so it can hide behind the MMAs as long as an
// accumulator is free to go on: two of 256 columns (or four of 128) fill TMEM.
#include <cuda_fp8.h>

#include "dtypes.cuh"
#include "tc_common.cuh"

namespace gsq {
namespace fp8 {

constexpr int kBlk = kFp8Block;

// ---------------------------------------------------------------------- quantization ---
// Rows: a half-warp per (row, block), eight values a lane, so a block's amax is four shuffles.
// One pass over x: bound by its bytes.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
quant_rows_kernel(const T* __restrict__ x, int64_t ld_x, int rows, int cols, int nblk,
                  uint8_t* __restrict__ codes, int64_t ld_c, float* __restrict__ scales,
                  int64_t ld_s) {
  const int sub = threadIdx.x & 15;
  const int64_t items = (int64_t)rows * nblk;
  const int64_t step = (int64_t)gridDim.x * 16;
  // both halves of a warp take the same number of turns (the shuffles are warp-wide)
  const int64_t first = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  const int64_t base = (int64_t)blockIdx.x * 16 + ((threadIdx.x >> 5) << 1);
  for (int64_t o = 0; base + o < items; o += step) {
    const int64_t it = first + o;
    const bool on = it < items;
    const int r = on ? (int)(it / nblk) : 0;
    const int b = on ? (int)(it - (int64_t)r * nblk) : 0;
    const int c = b * kBlk + sub * 8;
    float v[8];
    load8<T, VEC>(x + (int64_t)r * ld_x, c, on ? cols : 0, v);
    float a = amax8(v);
#pragma unroll
    for (int s = 8; s > 0; s >>= 1) a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, s));
    a = max_nan(a, kFp8AmaxMin);
    if (!on) continue;
    if (sub == 0) scales[(int64_t)b * ld_s + r] = __fdiv_rn(a, kFp8Max);
    const uint2 q = encode8(v, __fdiv_rn(kFp8Max, a));
    // the row pitch is a multiple of 16 bytes: the last vector of a row may run into its pad
    if (c < cols) *reinterpret_cast<uint2*>(codes + (int64_t)r * ld_c + c) = q;
  }
}

// A 128 x 128 tile per CTA, an 8 x 8 piece per thread (rows 8 (tid / 16).., columns
// 8 (tid % 16)..), in any of three forms from one read of the tile:
//   ROWS    a scale per row          -> codes [rows][ld_c], scales [cols / 128][ld_s]
//   COLS    a scale per column       -> codes_t [cols][ld_ct] (transposed through shared memory,
//                                       8 bytes a write), scales_t [rows / 128][ld_st]
//   BLOCKS  one scale for the tile   -> codes, scales [rows / 128][ld_s]
template <typename T, bool VEC, bool ROWS, bool COLS, bool BLOCKS>
__global__ void __launch_bounds__(256)
quant_tile_kernel(const T* __restrict__ x, int64_t ld_x, int rows, int cols,
                  uint8_t* __restrict__ codes, int64_t ld_c, float* __restrict__ scales,
                  int64_t ld_s, uint8_t* __restrict__ codes_t, int64_t ld_ct,
                  float* __restrict__ scales_t, int64_t ld_st) {
  __shared__ float red[8][kBlk];
  __shared__ __align__(16) uint8_t tile[COLS ? kBlk : 1][kBlk + 8];
  const int sub = threadIdx.x & 15, rg = threadIdx.x >> 4, warp = threadIdx.x >> 5;
  const int cb = blockIdx.x, rb = blockIdx.y;
  const int c = cb * kBlk + sub * 8, r0 = rb * kBlk + rg * 8;
  float v[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    load8<T, VEC>(x + (int64_t)(r0 + i < rows ? r0 + i : 0) * ld_x, c, r0 + i < rows ? cols : 0,
                  v[i]);
  if (ROWS) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float a = amax8(v[i]);
#pragma unroll
      for (int s = 8; s > 0; s >>= 1) a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, s));
      a = max_nan(a, kFp8AmaxMin);
      if (r0 + i < rows) {
        if (sub == 0) scales[(int64_t)cb * ld_s + r0 + i] = __fdiv_rn(a, kFp8Max);
        if (c < cols)
          *reinterpret_cast<uint2*>(codes + (int64_t)(r0 + i) * ld_c + c) =
              encode8(v[i], __fdiv_rn(kFp8Max, a));
      }
    }
  }
  if (COLS || BLOCKS) {
    float a[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      a[j] = fabsf(v[0][j]);
#pragma unroll
      for (int i = 1; i < 8; ++i) a[j] = max_nan(a[j], fabsf(v[i][j]));
      a[j] = max_nan(a[j], __shfl_xor_sync(0xffffffffu, a[j], 16));
    }
    if ((threadIdx.x & 16) == 0) {
#pragma unroll
      for (int j = 0; j < 8; ++j) red[warp][sub * 8 + j] = a[j];
    }
    __syncthreads();
    if (COLS) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float m = kFp8AmaxMin;
#pragma unroll
        for (int w = 0; w < 8; ++w) m = max_nan(m, red[w][sub * 8 + j]);
        if (rg == 0 && c + j < cols) scales_t[(int64_t)rb * ld_st + c + j] = __fdiv_rn(m, kFp8Max);
        float col[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) col[i] = v[i][j];
        *reinterpret_cast<uint2*>(&tile[sub * 8 + j][rg * 8]) = encode8(col, __fdiv_rn(kFp8Max, m));
      }
      __syncthreads();
      for (int e = threadIdx.x; e < kBlk * 16; e += 256) {
        const int cc = e >> 4, rr = (e & 15) * 8;
        if (cb * kBlk + cc < cols && rb * kBlk + rr < rows)
          *reinterpret_cast<uint2*>(codes_t + (int64_t)(cb * kBlk + cc) * ld_ct + rb * kBlk + rr) =
              *reinterpret_cast<const uint2*>(&tile[cc][rr]);
      }
    }
    if (BLOCKS) {
      float m = kFp8AmaxMin;
#pragma unroll
      for (int w = 0; w < 8; ++w)
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max_nan(m, red[w][sub * 8 + j]);
#pragma unroll
      for (int s = 8; s > 0; s >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, s));
      if (threadIdx.x == 0) scales[(int64_t)rb * ld_s + cb] = __fdiv_rn(m, kFp8Max);
      const float r = __fdiv_rn(kFp8Max, m);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (r0 + i < rows && c < cols)
          *reinterpret_cast<uint2*>(codes + (int64_t)(r0 + i) * ld_c + c) = encode8(v[i], r);
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

__device__ __forceinline__ void umma_e4m3(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
}

template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t* r) {
  if constexpr (N == 32) {
    tc::tmem_ld32_nowait(taddr, r);
  } else {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
        "%11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
  }
}

__device__ __forceinline__ void copy4(float* to, const float* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(tc::smem_u32(to)), "l"(from)
               : "memory");
}

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
// write, and sums into what is there).
template <typename T, int CW>
__device__ __forceinline__ void store_row(const GemmArgs& p, int m, int n0, const F2* acc) {
  if (m >= p.M) return;
  T* o = reinterpret_cast<T*>(p.out) + (int64_t)m * p.ld_o + n0;
#pragma unroll
  for (int c = 0; c < CW; ++c) {
    const float v = c & 1 ? acc[c >> 1].y : acc[c >> 1].x;
    if (n0 + c < p.N) o[c] = from_f32<T>(p.accumulate ? v + to_f32(o[c]) : v);
  }
}

// The tile's rows of one warp as boxes of 32 rows x 128 bytes, staged in shared memory in the
// store's 128-byte swizzle (16-byte chunk c of row r at c ^ (r % 8): a lane writes its own row
// without bank conflicts) and written by the TMA unit, which clips what lies outside the
// output. Two buffers a warp: a box is written while the last one is still being read.
template <typename T, int CW>
__device__ __forceinline__ void store_boxes(const GemmArgs& p, uint8_t* stage, int& buf, int lane,
                                            int m0, int n0, const F2* acc) {
  constexpr int BW = 128 / sizeof(T);  // columns of a box
  if (m0 >= p.M) return;
#pragma unroll
  for (int c0 = 0; c0 < CW; c0 += BW) {
    if (n0 + c0 < p.N) {
      uint8_t* b = stage + buf * 4096;
      if (lane == 0) tc::bulk_wait_read<1>();
      __syncwarp();
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        uint4 v;
        if constexpr (sizeof(T) == 2) {
          const F2* a = acc + (c0 + c * 8) / 2;
          v = make_uint4(f2_pack<T>(a[0]), f2_pack<T>(a[1]), f2_pack<T>(a[2]), f2_pack<T>(a[3]));
        } else {
          const F2* a = acc + (c0 + c * 4) / 2;
          v = make_uint4(__float_as_uint(a[0].x), __float_as_uint(a[0].y),
                         __float_as_uint(a[1].x), __float_as_uint(a[1].y));
        }
        *reinterpret_cast<uint4*>(b + lane * 128 + ((c ^ (lane & 7)) << 4)) = v;
      }
      tc::fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) {
        tma_store_2d(&p.o, b, n0 + c0, m0);
        tc::bulk_commit();
      }
      buf ^= 1;
    }
  }
}

// Register split of the wide kernel: 12 warps are launched with 168 registers a thread; warps
// 0-3 give theirs up to 72 and the epilogue's two warpgroups take 216 (128 x 72 + 256 x 216 =
// 384 x 168), enough for 128 sums and two groups of 32 accumulator columns in flight.
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
template <int BN, bool BROWS>
__global__ void __launch_bounds__(kThreads, 1) gemm_kernel(const __grid_constant__ GemmArgs p,
                                                           int dtype) {
  constexpr int kSlots = kTmemCols / BN;
  constexpr uint32_t kStage = (kBM + BN) * kBlk;
  constexpr int kStages = kPipeBytes / kStage;
  constexpr int CW = BN / 2;  // columns per epilogue warp
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages], tfull[4], tempty[4], last;
  __shared__ uint32_t tmem_base;
  constexpr int CH = BN == 256 ? 16 : 32;
  // k-blocks whose scales are on their way, and the ring's entries
  constexpr int kAhead = BROWS && BN == 256 ? 2 : 4, kRing = kAhead + 1;
  constexpr int kRow = 32 + (BROWS ? CW : 4);   // a k-block's scales of a warp: rows, columns
  __shared__ __align__(16) float ring_s[kEpiWarps][kRing * kRow];
  uint8_t* stage = smem + kStages * kStage;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      tc::mbar_init(&full[i], 1);
      tc::mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < kSlots; ++i) {
      tc::mbar_init(&tfull[i], 1);
      tc::mbar_init(&tempty[i], kEpiWarps);
    }
    tc::mbar_init(&last, 1);
    tc::fence_barrier_init();
  }
  if (warp == 1) tc::tmem_alloc(&tmem_base, kTmemCols);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = tmem_base;
  const int tiles = p.mt * p.nt;

  if (warp < 4) {
    if (BN == 256) regs_dec<72>();
    if (warp == 0 && lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
        int m, n;
        tile_at(p, t, m, n);
        for (int k = 0; k < p.kb; ++k, ++it) {
          const int s = it % kStages;
          if (it >= kStages && !tc::mbar_wait(&empty[s], (it / kStages - 1) & 1, p.err, 1)) {
            ok = false;
            break;
          }
          uint8_t* st = smem + s * kStage;
          tc::mbar_arrive_expect_tx(&full[s], kStage);
          tc::tma_load_2d(st, &p.a, &full[s], k * kBlk, m * kBM);
          tc::tma_load_2d(st + kBM * kBlk, &p.b, &full[s], k * kBlk, n * BN);
        }
      }
      // a copy still in flight after a timeout must land before the CTA's memory goes
      if (!ok)
        for (uint32_t i = it > kStages ? it - kStages : 0; i < it; ++i)
          tc::mbar_wait(&full[i % kStages], (i / kStages) & 1, nullptr, 0);
    } else if (warp == 1 && lane == 0) {
      constexpr uint32_t id = idesc_e4m3(kBM, BN);
      uint32_t it = 0;
      bool ok = true;
      for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
        for (int k = 0; k < p.kb; ++k, ++it) {
          const int s = it % kStages, sl = it % kSlots;
          if ((it >= kSlots && !tc::mbar_wait(&tempty[sl], (it / kSlots - 1) & 1, p.err, 2)) ||
              !tc::mbar_wait(&full[s], (it / kStages) & 1, p.err, 3)) {
            ok = false;
            break;
          }
          tc::fence_after_sync();
          const uint32_t a = tc::smem_u32(smem + s * kStage);
          const uint64_t da = tc::umma_desc_k_sw128(a),
                         db = tc::umma_desc_k_sw128(a + kBM * kBlk);
#pragma unroll
          for (int j = 0; j < 4; ++j)  // 32 values (32 bytes) of k per instruction
            umma_e4m3(tmem + sl * BN, da + 2 * j, db + 2 * j, id, j > 0);
          tc::umma_commit(&empty[s]);
          tc::umma_commit(&tfull[sl]);
        }
      }
      tc::umma_commit(&last);
      tc::mbar_wait(&last, 0, p.err, 4);
    }
  } else {
    if (BN == 256) regs_inc<216>();
    const int q = warp & 3, half = (warp - 4) >> 2;
    const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16) + half * CW;
    // The scales of the k-block kAhead ahead (of the next tile's, at a tile's end) are copied to
    // the warp's ring while this one is folded: a load from L2 takes longer than a k-block.
    float* ring = ring_s[warp - 4];
    int pt = blockIdx.x, pk = 0, pslot = 0, pn = 0;
    const float *psa = nullptr, *psb = nullptr;
    auto prefetch = [&]() {
      if (pt < tiles) {
        if (pk == 0) {
          int mi, ni;
          tile_at(p, pt, mi, ni);
          const int m = mi * kBM + q * 32 + lane;
          psa = p.sa + (m < p.M ? m : 0);
          pn = ni * BN + half * CW;
          // CW is 64 or 128 and pn a multiple of it: a warp's columns lie in one weight block
          psb = BROWS ? p.sb + lane : p.sb + min(pn, p.N - 1) / kBlk * p.sb_n;
        }
        float* to = ring + pslot * kRow;
        copy4(to + lane, psa);
        if (BROWS) {
#pragma unroll
          for (int i = 0; i < CW / 32; ++i)
            copy4(to + 32 + 32 * i + lane, psb + (pn + 32 * i + lane < p.N ? pn + 32 * i : -lane));
        } else if (lane == 0) {
          copy4(to + 32, psb);
        }
        psa += p.ld_sa;
        psb += p.sb_k;
        if (++pk == p.kb) {
          pk = 0;
          pt += gridDim.x;
        }
        pslot = pslot + 1 == kRing ? 0 : pslot + 1;
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) prefetch();
    uint32_t it = 0;
    int buf = 0, islot = 0;
    bool ok = true;
    for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
      int mi, ni;
      tile_at(p, t, mi, ni);
      const int m = mi * kBM + q * 32 + lane, n0 = ni * BN + half * CW;
      F2 acc[CW / 2];
#pragma unroll
      for (int c = 0; c < CW / 2; ++c) acc[c] = f2_same(0.f);
      for (int k = 0; k < p.kb; ++k, ++it) {
        const int sl = it % kSlots;
        asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
        ok = tc::mbar_wait(&tfull[sl], (it / kSlots) & 1, p.err, 5);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        __syncwarp();   // the other lanes' copies
        tc::fence_after_sync();
        const float* sc = ring + islot * kRow;
        islot = islot + 1 == kRing ? 0 : islot + 1;
        const float s = BROWS ? sc[lane] : sc[lane] * sc[32];
        const float* sbw = sc + 32;
        // CH columns are folded while the next are on their way from TMEM; the accumulator is
        // given back before the last ones are folded
        uint32_t r[2][CH];
        tmem_ld<CH>(lanes + sl * BN, r[0]);
#pragma unroll
        for (int c = 0; c < CW / CH; ++c) {
          tc::tmem_wait_ld();
          if (c + 1 < CW / CH) {
            tmem_ld<CH>(lanes + sl * BN + CH * (c + 1), r[(c + 1) & 1]);
          } else {
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&tempty[sl]);
          }
          const uint32_t* d = r[c & 1];
#pragma unroll
          for (int j = 0; j < CH / 2; ++j) {
            F2 v = {__uint_as_float(d[2 * j]), __uint_as_float(d[2 * j + 1])};
            if (BROWS) v = f2_mul(v, *reinterpret_cast<const F2*>(sbw + (BROWS ? CH * c + 2 * j : 0)));
            F2& to = acc[CH / 2 * c + j];
            to = f2_fma(v, f2_same(s), to);
          }
        }
        __syncwarp();   // (BROWS: every lane has read the ring's entry)
        prefetch();
      }
      if (ok) {
        uint8_t* st = stage + (warp - 4) * 8192;
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
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  if (warp == 1) tc::tmem_dealloc(tmem, kTmemCols);
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

template <int BN, bool BROWS>
static int launch_gemm(GemmArgs& p, int dtype, cudaStream_t st) {
  constexpr uint32_t kStage = (kBM + BN) * kBlk;
  constexpr uint32_t smem = kPipeBytes / kStage * kStage + kStageBytes + 1024;
  auto kern = gemm_kernel<BN, BROWS>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) !=
      cudaSuccess)
    return GSQ_ECUDA;
  if (BN == 256) {
    // the split above is only right for the register count it was made for
    cudaFuncAttributes at;
    if (cudaFuncGetAttributes(&at, kern) != cudaSuccess) return GSQ_ECUDA;
    if (at.numRegs != kLaunchRegs) return GSQ_ENOTSUP;
  }
  p.mt = (p.M + kBM - 1) / kBM;
  p.nt = (p.N + BN - 1) / BN;
  p.group = 16;
  const int64_t tiles = (int64_t)p.mt * p.nt;
  if (tiles > INT32_MAX / 2) return GSQ_EINVAL;
  const int grid = (int)(tiles < num_sms() ? tiles : num_sms());
  kern<<<grid, kThreads, smem, st>>>(p, dtype);
  GSQ_CHECK_LAUNCH();
  return GSQ_OK;
}

template <typename T>
static int quant_launch(const T* x, int rows, int cols, int64_t ld_x, uint8_t* codes, int64_t ld_c,
                        float* scales, int64_t ld_s, uint8_t* codes_t, int64_t ld_ct,
                        float* scales_t, int64_t ld_st, bool blocks, cudaStream_t st) {
  const bool vec = (uintptr_t)x % 16 == 0 && ld_x * sizeof(T) % 16 == 0;
  const int cb = (cols + kBlk - 1) / kBlk, rb = (rows + kBlk - 1) / kBlk;
  if (!blocks && !codes_t) {
    const int64_t items = (int64_t)rows * cb;
    int64_t g = (items + 15) / 16;
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
  return M > 0 && N > 0 && K > 0 && codes_ok(a, lda, K) && codes_ok(b, ldb, K) && sa &&
         ld_sa >= M && sb && sb_n >= 0 && sb_k >= 0 && out && dtype >= 0 && dtype <= 2 &&
         ld_out >= N && err && (uintptr_t)out % dtype_size(dtype) == 0 &&
         !(accumulate && dtype != F32) && !(sb_rows && sb_k < N);
}

inline bool quant_ok(const void* x, int dtype, int rows, int cols, int64_t ld_x) {
  return x && dtype >= 0 && dtype <= 2 && rows > 0 && cols > 0 && ld_x >= cols &&
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
  if (codes_t && (rows + 127) / 128 > 65535) return GSQ_EINVAL;
  return fp8::quant_any(x, dtype, rows, cols, ld_x, codes, ld_codes, scales, ld_scales, codes_t,
                        ld_codes_t, scales_t, ld_scales_t, false, (cudaStream_t)stream);
}

extern "C" int gsq_fp8_quant_blocks(const void* w, int dtype, int N, int K, int64_t ld_w,
                                    void* codes, int64_t ld_codes, float* scales,
                                    int64_t ld_scales, void* stream) {
  if (!fp8::quant_ok(w, dtype, N, K, ld_w) || !fp8::codes_ok(codes, ld_codes, K) || !scales ||
      ld_scales < (K + 127) / 128 || (N + 127) / 128 > 65535)
    return GSQ_EINVAL;
  return fp8::quant_any(w, dtype, N, K, ld_w, codes, ld_codes, scales, ld_scales, nullptr, 0,
                        nullptr, 0, true, (cudaStream_t)stream);
}

extern "C" int gsq_fp8_dequant(const void* codes, int64_t ld_codes, const float* scales,
                               int64_t ld_scales, int N, int K, void* out, int dtype,
                               int64_t ld_out, void* stream) {
  if (!fp8::codes_ok(codes, ld_codes, K) || !scales || N <= 0 || K <= 0 ||
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

extern "C" int gsq_fp8_gemm(int M, int N, int K, const void* a, int64_t lda, const float* sa,
                            int64_t ld_sa, const void* b, int64_t ldb, const float* sb,
                            int sb_rows, int64_t sb_n, int64_t sb_k, void* out,
                            int dtype, int64_t ld_out, int accumulate, int* err, void* stream) {
  if (!fp8::gemm_ok(M, N, K, a, lda, sa, ld_sa, b, ldb, sb, sb_rows, sb_n, sb_k, out, dtype, ld_out,
                    accumulate, err))
    return GSQ_EINVAL;
  fp8::GemmArgs p;
  // Tile width by the rounds that the busiest CTA walks: a 256-wide tile costs two 128-wide ones
  // but loads its A rows once (4094 x 896 x 4864: 128 wide tiles are one round of 148 SMs, 224
  // narrow ones two halves; 4864 x 896 x 4094: 152 wide tiles are two rounds, 266 narrow ones two
  // halves).
  const int64_t mt = (M + 127) / 128;
  const auto rounds = [&](int bn) { return (mt * ((N + bn - 1) / bn) + num_sms() - 1) / num_sms(); };
  const bool wide = 2 * rounds(256) <= rounds(128) + (rounds(128) >= 8 ? 1 : 0);
  if (!fp8::codes_map(&p.a, a, M, K, lda, fp8::kBM) ||
      !fp8::codes_map(&p.b, b, N, K, ldb, wide ? 256 : 128))
    return GSQ_ECUDA;
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
  if (sb_rows) return wide ? fp8::launch_gemm<256, true>(p, dtype, st)
                           : fp8::launch_gemm<128, true>(p, dtype, st);
  return wide ? fp8::launch_gemm<256, false>(p, dtype, st)
              : fp8::launch_gemm<128, false>(p, dtype, st);
}

extern "C" int gsq_fp8_linear(const void* x, int dtype, int M, int K, int64_t ld_x,
                              const void* codes, int64_t ld_codes, const float* scales,
                              int64_t ld_scales, int N, void* y, int y_dtype, int64_t ld_y,
                              void* workspace, int64_t workspace_bytes, int* err, void* stream) {
  if (M <= 0 || K <= 0 || N <= 0 || !workspace || (uintptr_t)workspace % 16) return GSQ_EINVAL;
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
  return gsq_fp8_gemm(M, N, K, q, ld_q, sq, M, codes, ld_codes, scales, 0, ld_scales, 1, y,
                      y_dtype, ld_y, 0, err, stream);
}
