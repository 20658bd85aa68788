// RMS norms before and after a block, fused with the block's gate, residual scale and sum:
//   n  = y r1 a,             r1 = (mean y^2 + eps)^-1/2,   a = w_post + offset   (y itself without w_post)
//   h' = h + alpha g n                                      (g = 1 without a gate)
//   x  = h' r2 b,            r2 = (mean h'^2 + eps)^-1/2,  b = w_pre + offset    (optional)
// in float32 from the unrounded h', each output rounded once; x also as e4m3 rows with a scale
// per 128 columns (the operand of the 8-bit product, without a bf16 copy in between).
// Vector-Jacobian product for the cotangents D of h' and X of x, from h, y and the row
// statistics r1, r2 of the forward pass (h' is recomputed, not stored unrounded):
//   u = X b,  d = D + r2 (u - h' r2^2 mean(u h')),  dh = d
//   m = alpha g d,  v = m a,  dy = r1 (v - y r1^2 mean(v y))
//   dw_post = sum m y r1,  dw_pre = sum X h' r2,  dg = sum alpha d n      (over rows, float32)
// With p = d y r1 the three parameter sums come from one: S = sum p over the rows of one gate row,
//   dg = alpha a S,  dw_post = sum over gate rows of alpha g S.
// Both directions are one pass over their rows, held in registers by a team of threads (a warp
// up to 256 columns, a block above: eight columns a thread), so they should be bound by the bytes
// of the rows. Rows that start on 16 bytes are read in fours of neighbouring columns; others
// column by column with the columns dealt round the team, which keeps every access of a warp one
// segment (neighbouring columns a thread would touch each sector several times).
// Measured: 16384 x 896 bf16 into e4m3 rows 31 us (3.3 TB/s, an instruction issued on 70 % of the
// schedulers' cycles), its gradient with a gate 50 us (3.5 TB/s, 55 %), the gradient of 6141 x 5121
// float16, column by column, 157 us. The gradient of 16384 x 896 reaches 73 % of the copy rate in
// float32 (73 us) and 54 % in bf16: what bounds the 16-bit forms is the instructions of a column and
// the barriers of a row's sums, not the bytes.
// Above 8192 columns the rows do not fit shared memory and a thread's 16 or 32 columns do not fit 64
// registers: the gradient spills 290 to 1700 bytes a thread (2048 x 32768 bf16: 711 us, 1.1 TB/s),
// the forward pass up to 600 (156 us, 3.5 TB/s).
// The column sums of the backward pass: each team adds its rows in registers and writes one
// partial row; a second kernel adds the partials in a fixed order (no atomics: the same inputs
// give the same bits).
#include "dtypes.cuh"
#include "tc_common.cuh"

namespace gsq {
namespace norm {

struct Fwd {
  const void *h, *y, *w_post, *w_pre, *gate;
  int64_t ld_h, ld_y;
  int T, H, per_gate;  // rows per row of the gate
  float alpha, eps, offset;
  void* h_out;
  int64_t ld_ho;
  void* x;
  int64_t ld_x;
  uint8_t* codes;
  int64_t ld_c;
  float* scales;
  int64_t ld_s;
  float* stats;  // [2][T] r1, r2
};

constexpr int kArrays = 4;  // y, h, dx, dh2
struct Bwd {
  const void* in[kArrays];  // dx NULL without w_pre, dh2 NULL for zeros
  int64_t ld[kArrays];
  const void *w_post, *w_pre, *gate;
  const float* stats;
  int T, H, per_gate;
  float alpha, offset;
  void *dh, *dy;
  int64_t ld_dh, ld_dy;
  int groups, splits;  // gate rows, and the parts each one's rows are cut into
  float* part_w;       // [teams][2][H] partials of dw_post, dw_pre
  float* part_g;       // [groups * splits][H] partials of dgate (dgate itself if splits == 1)
  int slots;           // rows in flight per team
  uint32_t row_bytes;  // shared memory of one array's row
  int* err;
};

// Sum over a row's team: a warp, or a block of up to 32 warps, whose two staging rows alternate
// so that one barrier per sum is enough. `red` is zero behind the block's warps.
template <bool WARP>
__device__ __forceinline__ float team_sum(float v, float (*red)[32], int& turn) {
  v = warp_sum(v);
  if (WARP) return v;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
  float* r = red[turn & 1];
  ++turn;
  if (lane == 0) r[warp] = v;
  __syncthreads();
  if (nw <= 8) {
    const float4 a = *reinterpret_cast<const float4*>(r), b = *reinterpret_cast<const float4*>(r + 4);
    return ((a.x + a.y) + (a.z + a.w)) + ((b.x + b.y) + (b.z + b.w));
  }
  return warp_sum(r[lane]);
}

template <typename T, bool VEC, bool PAD>
__device__ __forceinline__ void get4(const T* row, int q, int t, int tpr, int H, F2 v[2]) {
  pairs<T, VEC>(raw4<T, VEC, PAD>(row, q, t, tpr, H), v);
}

template <typename T, bool VEC>
__device__ __forceinline__ void put4(T* __restrict__ row, int q, int t, int tpr, int H,
                                     const F2 v[2]) {
  const int c0 = column<VEC>(q, 0, t, tpr);
  if constexpr (VEC) {
    if (c0 < H) {
      if constexpr (sizeof(T) == 2)
        *reinterpret_cast<uint2*>(row + c0) = make_uint2(f2_pack<T>(v[0]), f2_pack<T>(v[1]));
      else
        *reinterpret_cast<float4*>(row + c0) = make_float4(v[0].x(), v[0].y(), v[1].x(), v[1].y());
    }
  } else {
    const float f[4] = {v[0].x(), v[0].y(), v[1].x(), v[1].y()};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c0 + j * tpr < H) row[c0 + j * tpr] = from_f32<T>(f[j]);
  }
}

__device__ __forceinline__ float f2_dot(const F2 a[2], const F2 b[2]) {
  const F2 s = f2_fma(a[1], b[1], f2_mul(a[0], b[0]));
  return s.x() + s.y();
}
__device__ __forceinline__ float f2_at(const F2 v[2], int j) {
  return j & 1 ? v[j >> 1].y() : v[j >> 1].x();
}

// 1 / sqrt(m): the hardware's estimate (2 steps off at most) after one Newton iteration
// r += r (1 - m r^2) / 2, whose residual is formed in one fused operation.
__device__ __forceinline__ float inv_root(float m) {
  const float r = rsqrtf(m);
  const float n = fmaf(0.5f * r, fmaf(-m * r, r, 1.f), r);
  return isfinite(n) ? n : r;   // (m = infinity or denormal: the estimate itself)
}

// A thread's columns of the parameters: alpha a g (from the gate row g) and b; 1 stands for a
// missing w_post or gate, 0 for a missing w_pre.
struct Params {
  const void *w_post, *w_pre, *gate;
  float alpha, offset;
  int H;
};

template <typename T, bool VEC>
struct Columns {
  const Params& p;
  int t, tpr;
  __device__ __forceinline__ void a(int q, F2 v[2]) const {
    if (p.w_post) get4<T, VEC, false>(reinterpret_cast<const T*>(p.w_post), q, t, tpr, p.H, v);
#pragma unroll
    for (int j = 0; j < 2; ++j) v[j] = p.w_post ? f2_add(v[j], f2_same(p.offset)) : f2_same(1.f);
  }
  __device__ __forceinline__ void alpha_g(int g, int q, F2 v[2]) const {
    if (p.gate)
      get4<T, VEC, false>(reinterpret_cast<const T*>(p.gate) + (int64_t)g * p.H, q, t, tpr, p.H, v);
#pragma unroll
    for (int j = 0; j < 2; ++j) v[j] = p.gate ? f2_mul(v[j], f2_same(p.alpha)) : f2_same(p.alpha);
  }
  __device__ __forceinline__ void alpha_ag(int g, int q, F2 v[2]) const {
    F2 gv[2];
    a(q, v);
    alpha_g(g, q, gv);
#pragma unroll
    for (int j = 0; j < 2; ++j) v[j] = f2_mul(v[j], gv[j]);
  }
  __device__ __forceinline__ void b(int q, F2 v[2]) const {
    if (p.w_pre) get4<T, VEC, false>(reinterpret_cast<const T*>(p.w_pre), q, t, tpr, p.H, v);
#pragma unroll
    for (int j = 0; j < 2; ++j) v[j] = p.w_pre ? f2_add(v[j], f2_same(p.offset)) : f2_same(0.f);
  }
};

// Persistent teams: team i takes rows i, i + teams, ...; the parameters' columns stay in
// registers (HOLD) where the team leaves room for them, and the next row's loads are issued
// before this row is worked on (16384 x 896 into e4m3 rows: 44 us before the two, 35 with
// them).
template <typename T, bool VEC, bool WARP, int Q, bool HOLD, bool FP8, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) fwd_kernel(const __grid_constant__ Fwd p) {
  __shared__ __align__(16) float red[2][32];
  __shared__ uint32_t amax_s[FP8 && !VEC ? 512 : 1];   // two rows' blocks, in turn
  int turn = 0;
  const int t = WARP ? threadIdx.x & 31 : threadIdx.x, tpr = WARP ? 32 : blockDim.x;
  const int w = WARP ? threadIdx.x >> 5 : 0;
  const int teams = WARP ? gridDim.x * 8 : gridDim.x;
  if (!WARP && threadIdx.x < 64) red[threadIdx.x >> 5][threadIdx.x & 31] = 0.f;
  if (FP8 && !VEC)
    for (int i = threadIdx.x; i < 512; i += blockDim.x) amax_s[i] = 0u;
  __syncthreads();
  const Params pa = {p.w_post, p.w_pre, p.gate, p.alpha, p.offset, p.H};
  const Columns<T, VEC> col{pa, t, tpr};
  const float inv_H = 1.f / (float)p.H;
  const T* h_in = reinterpret_cast<const T*>(p.h);
  const T* y_in = reinterpret_cast<const T*>(p.y);
  F2 ag[HOLD ? Q : 1][2], bw[HOLD ? Q : 1][2];
  int held = -1;
  int row = WARP ? blockIdx.x * 8 + w : blockIdx.x;
  Four<T> yn[Q], hn[Q];   // the next row
  auto load = [&](int r) {
#pragma unroll
    for (int q = 0; q < Q; ++q) yn[q] = raw4<T, VEC, false>(y_in + (int64_t)r * p.ld_y, q, t, tpr, p.H);
#pragma unroll
    for (int q = 0; q < Q; ++q) hn[q] = raw4<T, VEC, false>(h_in + (int64_t)r * p.ld_h, q, t, tpr, p.H);
  };
  int half = 0;
  if (HOLD && row < p.T) load(row);
  for (; row < p.T; row += teams, half ^= 256) {
    F2 y[Q][2], h[Q][2];
    if (!HOLD) load(row);
#pragma unroll
    for (int q = 0; q < Q; ++q) pairs<T, VEC>(yn[q], y[q]), pairs<T, VEC>(hn[q], h[q]);
    if (HOLD && row + teams < p.T) load(row + teams);
    const int g = p.gate ? row / p.per_gate : 0;
    if (HOLD && g != held) {
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        col.alpha_ag(g, q, ag[HOLD ? q : 0]);
        if (held < 0) col.b(q, bw[HOLD ? q : 0]);
      }
      held = g;
    }
    float r1 = 1.f, r2 = 1.f;
    if (p.w_post) {
      float s = 0.f;
#pragma unroll
      for (int q = 0; q < Q; ++q) s += f2_dot(y[q], y[q]);
      r1 = inv_root(fmaf(team_sum<WARP>(s, red, turn), inv_H, p.eps));
    }
    float s = 0.f;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      F2 v[2];
      if (!HOLD) col.alpha_ag(g, q, v);
#pragma unroll
      for (int j = 0; j < 2; ++j)
        h[q][j] = f2_fma(HOLD ? ag[HOLD ? q : 0][j] : v[j], f2_mul(y[q][j], f2_same(r1)), h[q][j]);
      s += f2_dot(h[q], h[q]);
      if (p.h_out)
        put4<T, VEC>(reinterpret_cast<T*>(p.h_out) + (int64_t)row * p.ld_ho, q, t, tpr, p.H, h[q]);
    }
    if (p.w_pre) {
      r2 = inv_root(fmaf(team_sum<WARP>(s, red, turn), inv_H, p.eps));
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        F2 v[2];
        if (!HOLD) col.b(q, v);
#pragma unroll
        for (int j = 0; j < 2; ++j)
          h[q][j] = f2_mul(f2_mul(h[q][j], f2_same(r2)), HOLD ? bw[HOLD ? q : 0][j] : v[j]);
        if (!FP8)
          put4<T, VEC>(reinterpret_cast<T*>(p.x) + (int64_t)row * p.ld_x, q, t, tpr, p.H, h[q]);
      }
      if (FP8 && VEC) {
        // a warp's chunk is one 128-column block; magnitudes compare as their bits (NaN is above
        // infinity). Lane 2 q divides m / 448, lane 2 q + 1 448 / m.
        const int lane = t & 31;
        float num = 1.f, den = 1.f;
#pragma unroll
        for (int q = 0; q < Q; ++q) {
          const uint32_t bits = amax4(h[q]);
          const float m = max_nan(__uint_as_float(__reduce_max_sync(0xffffffffu, bits)),
                                  kFp8AmaxMin);
          if (lane == 2 * q) num = m, den = kFp8Max;
          if (lane == 2 * q + 1) num = kFp8Max, den = m;
        }
        const float quot = __fdiv_rn(num, den);
#pragma unroll
        for (int q = 0; q < Q; ++q) {
          const float r = __shfl_sync(0xffffffffu, quot, 2 * q + 1);
          const int c0 = column<true>(q, 0, t, tpr);
          if (lane == 2 * q && c0 - 8 * q < p.H)   // (the warp's first column of the chunk)
            p.scales[(int64_t)(c0 / kFp8Block) * p.ld_s + row] = quot;
          put_codes<true>(p.codes + (int64_t)row * p.ld_c, q, t, tpr, p.H, encode4(h[q], r));
        }
      }
      if (FP8 && !VEC) {
        // a warp's 32 columns of one j lie in one block: a warp maximum, then one shared-memory
        // maximum per warp and block
        const int nb = (p.H + kFp8Block - 1) / kFp8Block;
        uint32_t* am = amax_s + half + (WARP ? w * 4 : 0);
        uint32_t* other = amax_s + (half ^ 256) + (WARP ? w * 4 : 0);
#pragma unroll
        for (int q = 0; q < Q; ++q)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(fabsf(f2_at(h[q], j))));
            const int c = column<false>(q, j, t, tpr);
            if ((t & 31) == 0 && c < p.H) atomicMax(am + c / kFp8Block, m);
          }
        if (WARP) __syncwarp();
        else __syncthreads();
        for (int b = t; b < nb; b += tpr) {
          p.scales[(int64_t)b * p.ld_s + row] =
              __fdiv_rn(max_nan(__uint_as_float(am[b]), kFp8AmaxMin), kFp8Max);
          other[b] = 0u;   // for the next row
        }
#pragma unroll
        for (int q = 0; q < Q; ++q)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int c = column<false>(q, j, t, tpr);
            if (c < p.H) {
              const float m = max_nan(__uint_as_float(am[c / kFp8Block]), kFp8AmaxMin);
              p.codes[(int64_t)row * p.ld_c + c] = (uint8_t)cvt4_e4m3(
                  __fmul_rn(f2_at(h[q], j), __fdiv_rn(kFp8Max, m)), 0.f, 0.f, 0.f);
            }
          }
        // (a block's next row passes the barrier of its second sum before it adds to `other`)
        if (WARP) __syncwarp();
      }
    }
    if (t == 0) {
      p.stats[row] = r1;
      p.stats[p.T + row] = r2;
    }
  }
}

// The rows of a team, in order: items (a part of a gate row's rows) team, team + teams, ...
struct Rows {
  int item, row, hi;   // the item, and what is left of its rows; item -1: none
  __device__ __forceinline__ void open(const Bwd& p, int64_t i) {
    item = -1;
    if (i >= (int64_t)p.groups * p.splits) return;
    item = (int)i;
    const int g = item / p.splits, part = item - g * p.splits;
    row = (int)((int64_t)p.per_gate * part / p.splits) + g * p.per_gate;
    hi = (int)((int64_t)p.per_gate * (part + 1) / p.splits) + g * p.per_gate;
  }
  __device__ __forceinline__ void next(const Bwd& p, int teams) {
    if (++row == hi) open(p, (int64_t)item + teams);
  }
};

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes,
                                          uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          tc::smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(tc::smem_u32(bar))
      : "memory");
}

// Copies a row of array i into a slot (the team's thread i does): from the 16-byte boundary at or
// below its start to that at or above its end (the few bytes around a row that does not start or
// end there lie in the same 16 bytes as the row's own).
template <typename T>
__device__ __forceinline__ void fetch_row(const Bwd& p, int row, int i, uint8_t* slot,
                                          uint64_t* bar) {
  if (!p.in[i]) return;
  const uintptr_t s = (uintptr_t)(reinterpret_cast<const T*>(p.in[i]) + (int64_t)row * p.ld[i]);
  const uintptr_t lo = s & ~(uintptr_t)15, hi = (s + p.H * sizeof(T) + 15) & ~(uintptr_t)15;
  tc::mbar_arrive_expect_tx(bar, (uint32_t)(hi - lo));
  bulk_load(slot + i * p.row_bytes, reinterpret_cast<const void*>(lo), (uint32_t)(hi - lo), bar);
}

constexpr int kMaxSlots = 4;

// Where a thread's alpha a g and b are kept: in registers up to 768 threads a team, in shared
// memory up to 1024, and read anew for every row where a row does not fit shared memory.
enum Weights { W_REG, W_SMEM, W_MEM };

// Persistent teams, 4 Q columns a thread. Unless W_MEM, a team's rows arrive in shared memory by
// bulk copies, `slots` rows ahead, so that the loads run on through the two sums of a row, and
// dh2 is read only after the first of them: 6 of 8 registers a column.
// ALL: both norms and both cotangents are there.
template <typename T, bool VEC, bool WARP, int Q, int W, int THREADS, bool ALL>
__global__ void __launch_bounds__(THREADS, WARP ? 2 : 1) bwd_kernel(const __grid_constant__ Bwd p) {
  constexpr bool STAGED = W != W_MEM;
  constexpr int QW = W == W_REG ? Q : 1;
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ __align__(16) float red[2][32];
  __shared__ __align__(8) uint64_t bars[WARP ? 8 : 1][kMaxSlots];
  int turn = 0;
  const int w = WARP ? threadIdx.x >> 5 : 0, per = WARP ? blockDim.x >> 5 : 1;
  const int t = WARP ? threadIdx.x & 31 : threadIdx.x, tpr = WARP ? 32 : blockDim.x;
  const int team = blockIdx.x * per + w, teams = gridDim.x * per;
  const float inv_H = 1.f / (float)p.H;
  uint64_t* bar = bars[w];
  const uint32_t slot_bytes = kArrays * p.row_bytes;
  uint8_t* mine = dyn + (size_t)w * p.slots * slot_bytes;
  // W_SMEM: b and alpha a g
  const int room = 4 * Q * tpr;
  float* b_s = reinterpret_cast<float*>(dyn + (size_t)per * p.slots * slot_bytes);
  float* ag_s = b_s + room;
  if (!WARP && threadIdx.x < 64) red[threadIdx.x >> 5][threadIdx.x & 31] = 0.f;
  if (W == W_SMEM)
    for (int c = threadIdx.x; c < room; c += blockDim.x)
      b_s[c] = p.w_pre && c < p.H ? to_f32(reinterpret_cast<const T*>(p.w_pre)[c]) + p.offset : 0.f;
  if (STAGED && t == 0) {
    int arrays = 0;
#pragma unroll
    for (int i = 0; i < kArrays; ++i) arrays += p.in[i] != nullptr;
    for (int i = 0; i < p.slots; ++i) tc::mbar_init(&bar[i], arrays);
    tc::fence_barrier_init();
  }
  __syncthreads();
  Rows it, ahead;   // the row at work, and the next to fetch
  it.open(p, team);
  ahead = it;
  if (STAGED)
    for (int i = 0; i < p.slots && ahead.item >= 0; ++i, ahead.next(p, teams))
      if (t < kArrays) fetch_row<T>(p, ahead.row, t, mine + i * slot_bytes, &bar[i]);
  const bool post = ALL || p.w_post != nullptr, pre = ALL || p.w_pre != nullptr,
             cot = ALL || p.in[3] != nullptr;   // (the cotangent of h')
  const Params pa = {p.w_post, p.w_pre, p.gate, p.alpha, p.offset, p.H};
  const Columns<T, VEC> cols{pa, t, tpr};
  F2 S[Q][2], sw[Q][2];     // sums of d y r1 and of dx h' r2
  F2 ag[QW][2], bw[QW][2];
#pragma unroll
  for (int q = 0; q < Q; ++q)
#pragma unroll
    for (int j = 0; j < 2; ++j) S[q][j] = sw[q][j] = f2_same(0.f);
  int held = -1;   // the item whose alpha a g is held
  bool alive = true, opened = false;
  int slot = 0;
  uint32_t phase = 0;
  for (; it.item >= 0; it.next(p, teams)) {
    const int row = it.row;
    if (STAGED && it.item != held) {
      const int g = it.item / p.splits;
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        F2 v[2], u[2];
        cols.alpha_ag(g, q, v);
        if (W == W_REG) {
          cols.b(q, u);
#pragma unroll
          for (int j = 0; j < 2; ++j) ag[W == W_REG ? q : 0][j] = v[j], bw[W == W_REG ? q : 0][j] = u[j];
        } else {   // (each thread reads only what it wrote)
          put4<float, VEC>(ag_s, q, t, tpr, room, v);
        }
      }
      held = it.item;
    }
    const float r1 = post ? p.stats[row] : 1.f, r2 = pre ? p.stats[p.T + row] : 1.f;
    // (after a timeout the rows run on unread, so that the block's barriers keep their count)
    if (STAGED && alive) alive = tc::mbar_wait(&bar[slot], phase, p.err, 6);
    auto read = [&](int i, int q, F2 v[2]) {
      if (STAGED) {
        // (a row that does not start on 16 bytes lies that far into its copy)
        uint32_t off = i * p.row_bytes;
        if (!VEC)
          off += (uint32_t)(uintptr_t)(reinterpret_cast<const T*>(p.in[i]) + (int64_t)row * p.ld[i]) & 15u;
        get4<T, VEC, true>(reinterpret_cast<const T*>(mine + slot * slot_bytes + off), q, t, tpr,
                           p.H, v);
      } else {
        get4<T, VEC, false>(reinterpret_cast<const T*>(p.in[i]) + (int64_t)row * p.ld[i], q, t, tpr,
                            p.H, v);
      }
    };
    F2 y[Q][2], h[Q][2], u[Q][2];
    float s = 0.f;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      F2 wv[2];
      read(0, q, y[q]);
      read(1, q, h[q]);
      if (W == W_SMEM) get4<float, VEC, true>(ag_s, q, t, tpr, room, wv);
      if (W == W_MEM) cols.alpha_ag(it.item / p.splits, q, wv);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        y[q][j] = f2_mul(y[q][j], f2_same(r1));
        h[q][j] = f2_mul(f2_fma(W == W_REG ? ag[W == W_REG ? q : 0][j] : wv[j], y[q][j], h[q][j]),
                         f2_same(r2));   // h' r2
      }
      if (pre) {
        read(2, q, u[q]);
        if (W == W_SMEM) get4<float, VEC, true>(b_s, q, t, tpr, room, wv);
        if (W == W_MEM) cols.b(q, wv);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (!pre) u[q][j] = f2_same(0.f);
        sw[q][j] = f2_fma(u[q][j], h[q][j], sw[q][j]);
        if (pre) u[q][j] = f2_mul(u[q][j], W == W_REG ? bw[W == W_REG ? q : 0][j] : wv[j]);
      }
      s += f2_dot(u[q], h[q]);
    }
    const float mu = team_sum<WARP>(s, red, turn) * inv_H;
    s = 0.f;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      F2 wv[2], d[2], e[2];
      if (cot) read(3, q, d);
      if (W == W_SMEM) get4<float, VEC, true>(ag_s, q, t, tpr, room, wv);
      if (W == W_MEM) cols.alpha_ag(it.item / p.splits, q, wv);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (!cot) d[j] = f2_same(0.f);
        if (pre) d[j] = f2_fma(f2_same(r2), f2_fma(f2_same(-mu), h[q][j], u[q][j]), d[j]);
        e[j] = f2_mul(d[j], y[q][j]);
        S[q][j] = f2_add(S[q][j], e[j]);
        u[q][j] = f2_mul(W == W_REG ? ag[W == W_REG ? q : 0][j] : wv[j], d[j]);   // v
      }
      s += f2_dot(W == W_REG ? ag[W == W_REG ? q : 0] : wv, e);
      put4<T, VEC>(reinterpret_cast<T*>(p.dh) + (int64_t)row * p.ld_dh, q, t, tpr, p.H, d);
    }
    float mv = team_sum<WARP>(s, red, turn) * inv_H;
    if (!post) mv = 0.f;
    // every thread has read the slot (the sum's barrier; a warp's shuffles): the next row may land
    if (STAGED && ahead.item >= 0) {
      if (t < kArrays && alive)
        fetch_row<T>(p, ahead.row, t, mine + slot * slot_bytes, &bar[slot]);
      ahead.next(p, teams);
    }
    if (++slot == p.slots) {
      slot = 0;
      phase ^= 1;
    }
#pragma unroll
    for (int q = 0; q < Q; ++q) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
        u[q][j] = f2_mul(f2_same(r1), f2_fma(f2_same(-mv), y[q][j], u[q][j]));
      put4<T, VEC>(reinterpret_cast<T*>(p.dy) + (int64_t)row * p.ld_dy, q, t, tpr, p.H, u[q]);
    }
    if (row + 1 == it.hi) {
      const int g = it.item / p.splits;
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        F2 a[2], gv[2];
        cols.a(q, a);
        cols.alpha_g(g, q, gv);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int col = column<VEC>(q, j, t, tpr);
          if (col < p.H) {
            const float sj = f2_at(S[q], j);
            if (p.part_g) p.part_g[(int64_t)it.item * p.H + col] = p.alpha * f2_at(a, j) * sj;
            float* pw = p.part_w + (int64_t)team * 2 * p.H + col;
            const float v = f2_at(gv, j) * sj;
            *pw = opened ? *pw + v : v;
          }
        }
        S[q][0] = S[q][1] = f2_same(0.f);
      }
      opened = true;
    }
  }
#pragma unroll
  for (int q = 0; q < Q; ++q)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int col = column<VEC>(q, j, t, tpr);
      if (col < p.H) {
        p.part_w[((int64_t)team * 2 + 1) * p.H + col] = f2_at(sw[q], j);
        if (!opened) p.part_w[(int64_t)team * 2 * p.H + col] = 0.f;
      }
    }
  // (every copy issued was waited for, unless a wait gave up: then its last copies are)
  if (STAGED && !alive && t == 0)
    for (int i = 0; i < p.slots; ++i)
      for (int ph = 0; ph < 2; ++ph) tc::mbar_wait(&bar[i], ph, nullptr, 0);
}

// out[o][c] = sum over i < n of part[(o outer + i) stride + c]: a block takes 32 columns of one
// output row, 32 threads a column; the order of the sums does not depend on the launch.
struct Reduce {
  const float* part;
  float* out;
  int n;
  int64_t outer, stride;
};

__global__ void __launch_bounds__(1024)
reduce_kernel(Reduce r0, Reduce r1, Reduce r2, int H) {
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + lane;
  const int64_t o = blockIdx.y < 2 ? 0 : blockIdx.y - 2;
  const Reduce& r = blockIdx.y == 0 ? r0 : (blockIdx.y == 1 ? r1 : r2);
  if (!r.out) return;
  float a = 0.f;
  // eight loads in flight a thread, also where fewer are left
  for (int i0 = w; i0 < r.n; i0 += 256) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = i0 + 32 * j;
      v[j] = col < H && i < r.n ? r.part[(o * r.outer + i) * r.stride + col] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) a += v[j];
  }
  s[w][lane] = a;
  __syncthreads();
  a = warp_sum(s[lane][w]);
  const int c = blockIdx.x * 32 + w;
  if (lane == 0 && c < H) r.out[o * H + c] = a;
}

constexpr int kMaxH = 32768;

// Threads of a block team with Q chunks of four columns each.
inline int team_threads(int H, int q) { return ((H + 4 * q - 1) / (4 * q) + 31) / 32 * 32; }

template <typename T, bool VEC, bool WARP, int Q, bool HOLD, int THREADS>
static int fwd_launch(const Fwd& p, int threads, cudaStream_t st) {
  int64_t blocks = WARP ? ((int64_t)p.T + 7) / 8 : p.T;
  // the blocks that stay resident: 1024 threads of 64 registers an SM
  const int64_t most = (int64_t)num_sms() * (1024 / threads);
  if (blocks > most) blocks = most;
  const unsigned g = (unsigned)blocks;
  if (p.codes) fwd_kernel<T, VEC, WARP, Q, HOLD, true, THREADS><<<g, threads, 0, st>>>(p);
  else fwd_kernel<T, VEC, WARP, Q, HOLD, false, THREADS><<<g, threads, 0, st>>>(p);
  GSQ_CHECK_LAUNCH();
  return GSQ_OK;
}

template <typename T, bool VEC>
static int fwd_any(const Fwd& p, cudaStream_t st) {
  if (p.H <= 256) return fwd_launch<T, VEC, true, 2, true, 256>(p, 256, st);
  if (p.H <= 4096) return fwd_launch<T, VEC, false, 2, true, 512>(p, team_threads(p.H, 2), st);
  if (p.H <= 8192) return fwd_launch<T, VEC, false, 2, false, 1024>(p, team_threads(p.H, 2), st);
  if (p.H <= 16384) return fwd_launch<T, VEC, false, 4, false, 1024>(p, team_threads(p.H, 4), st);
  return fwd_launch<T, VEC, false, 8, false, 1024>(p, team_threads(p.H, 8), st);
}

// How the backward pass runs: as many teams as stay resident, the parts each gate row's rows
// are cut into so that the teams share them evenly, and the rows in flight per team.
struct Plan {
  bool warp;
  int q, threads, blocks, teams, splits, slots, weights;
  uint32_t row_bytes;
  size_t smem;
  int64_t ws;  // floats of workspace
};

constexpr size_t kSmemTeam = 200 * 1024;  // of an SM, shared by its teams

static Plan bwd_plan(int T, int H, int dtype, int groups, bool gate) {
  Plan pl;
  const bool warp = H <= 256;
  const int q = H <= 8192 ? 2 : (H <= 16384 ? 4 : 8);
  // warps of a block of warp teams: fewer where there are too few rows to give every SM eight
  int per = 1;
  if (warp) per = (int)((T + (int64_t)num_sms() - 1) / num_sms());
  if (per > 8) per = 8;
  pl.warp = warp;
  pl.q = q;
  pl.threads = warp ? 32 * per : team_threads(H, q);
  // room for the whole team's columns (a row is read past H) and for an unaligned start
  const int room = 4 * q * (warp ? 32 : pl.threads);
  pl.row_bytes = (uint32_t)(room * dtype_size(dtype) + 32);
  pl.weights = H <= 6144 ? W_REG : W_SMEM;
  const size_t slot = (size_t)kArrays * pl.row_bytes;
  const size_t fix = pl.weights == W_SMEM ? (size_t)8 * room : 0;
  if (q > 2 || slot + fix > kSmemTeam) pl.weights = W_MEM;
  // teams of an SM: 640 threads of 96 registers, or blocks of eight warp teams
  const int sm_blocks = warp ? 2 : (pl.weights == W_REG && pl.threads <= 640 ? 640 / pl.threads : 1);
  pl.slots = 1;
  pl.smem = 0;
  if (pl.weights != W_MEM) {
    const size_t fit = (kSmemTeam / sm_blocks - fix) / (slot * per);
    pl.slots = (int)(fit < 1 ? 1 : (fit > kMaxSlots ? kMaxSlots : fit));
    pl.smem = (size_t)pl.slots * slot * per + fix;
  }
  int64_t blocks = ((int64_t)T + per - 1) / per;
  const int64_t most = (int64_t)num_sms() * sm_blocks;
  if (blocks > most) blocks = most;
  pl.blocks = (int)blocks;
  pl.teams = pl.blocks * per;
  // one part a team at most: a part more than there are teams would take a second turn
  const int rows = T / groups;
  int s = pl.teams / groups;
  s = s < 1 ? 1 : (s > rows ? rows : s);
  pl.splits = s;
  pl.ws = (int64_t)pl.teams * 2 * H + (gate && s > 1 ? (int64_t)groups * s * H : 0);
  return pl;
}

template <typename T, bool VEC, bool WARP, int Q, int W, int THREADS>
static int bwd_launch(const Bwd& p, const Plan& pl, cudaStream_t st) {
  auto kern = p.w_post && p.w_pre && p.in[3] ? bwd_kernel<T, VEC, WARP, Q, W, THREADS, true>
                                             : bwd_kernel<T, VEC, WARP, Q, W, THREADS, false>;
  // The limit is the function's, for all host threads: one value for every call (bwd_plan gives no
  // team more), so that none lowers it between another's setting and launch.
  if (pl.smem > kSmemTeam) return GSQ_ENOTSUP;
  if (W != W_MEM &&
      cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemTeam) !=
          cudaSuccess)
    return GSQ_ECUDA;
  kern<<<pl.blocks, pl.threads, pl.smem, st>>>(p);
  GSQ_CHECK_LAUNCH();
  return GSQ_OK;
}

template <typename T, bool VEC>
static int bwd_any(const Bwd& p, const Plan& pl, cudaStream_t st) {
  if (pl.warp) return bwd_launch<T, VEC, true, 2, W_REG, 256>(p, pl, st);
  if (pl.weights == W_REG) return pl.threads <= 640
                                      ? bwd_launch<T, VEC, false, 2, W_REG, 640>(p, pl, st)
                                      : bwd_launch<T, VEC, false, 2, W_REG, 768>(p, pl, st);
  if (pl.weights == W_SMEM) return bwd_launch<T, VEC, false, 2, W_SMEM, 1024>(p, pl, st);
  if (pl.q == 2) return bwd_launch<T, VEC, false, 2, W_MEM, 1024>(p, pl, st);
  if (pl.q == 4) return bwd_launch<T, VEC, false, 4, W_MEM, 1024>(p, pl, st);
  return bwd_launch<T, VEC, false, 8, W_MEM, 1024>(p, pl, st);
}

inline bool row_vec(const void* p, int64_t ld, size_t es) {
  return !p || ((uintptr_t)p % 16 == 0 && ld * es % 16 == 0);
}

inline bool row_ok(const void* p, int64_t ld, int H, size_t es) {
  return p && ld >= H && (uintptr_t)p % es == 0;
}

}  // namespace norm
}  // namespace gsq

using namespace gsq;

extern "C" int gsq_residual_norm(const void* h, int64_t ld_h, const void* y, int64_t ld_y,
                                 const void* w_post, const void* w_pre, const void* gate,
                                 int gate_rows, int T, int H, int dtype, float alpha, float eps,
                                 float offset, void* h_out, int64_t ld_ho, void* x, int64_t ld_x,
                                 void* codes, int64_t ld_codes, float* scales, int64_t ld_scales,
                                 float* stats, void* stream) {
  if (T <= 0 || T > kMaxDim || H <= 0 || dtype < 0 || dtype > 2 || !stats) return GSQ_EINVAL;
  const size_t es = dtype_size(dtype);
  if (!norm::row_ok(h, ld_h, H, es) || !norm::row_ok(y, ld_y, H, es)) return GSQ_EINVAL;
  if (!lies_on(w_post, es) || !lies_on(w_pre, es) || !lies_on(gate, es) || !lies_on(stats, 4) ||
      !lies_on(scales, 4))
    return GSQ_EINVAL;
  if (gate && (gate_rows <= 0 || T % gate_rows)) return GSQ_EINVAL;
  if (h_out && !norm::row_ok(h_out, ld_ho, H, es)) return GSQ_EINVAL;
  if (w_pre ? (!x && !codes) || (x && codes) : x || codes) return GSQ_EINVAL;
  if (x && !norm::row_ok(x, ld_x, H, es)) return GSQ_EINVAL;
  if (codes && ((uintptr_t)codes % 16 || ld_codes % 16 || ld_codes < H || !scales ||
                ld_scales < T))
    return GSQ_EINVAL;
  if (!h_out && !w_pre) return GSQ_EINVAL;
  if (H > norm::kMaxH) return GSQ_ENOTSUP;
  norm::Fwd p;
  p.h = h; p.y = y; p.w_post = w_post; p.w_pre = w_pre; p.gate = gate;
  p.ld_h = ld_h; p.ld_y = ld_y;
  p.T = T; p.H = H; p.per_gate = gate ? T / gate_rows : T;
  p.alpha = alpha; p.eps = eps; p.offset = offset;
  p.h_out = h_out; p.ld_ho = ld_ho; p.x = x; p.ld_x = ld_x;
  p.codes = (uint8_t*)codes; p.ld_c = ld_codes; p.scales = scales; p.ld_s = ld_scales;
  p.stats = stats;
  const bool vec = H % 4 == 0 && norm::row_vec(h, ld_h, es) && norm::row_vec(y, ld_y, es) &&
                   norm::row_vec(w_post, 0, es) && norm::row_vec(w_pre, 0, es) &&
                   norm::row_vec(gate, H, es) && norm::row_vec(h_out, ld_ho, es) &&
                   norm::row_vec(x, ld_x, es);
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == BF16) return vec ? norm::fwd_any<__nv_bfloat16, true>(p, st)
                                : norm::fwd_any<__nv_bfloat16, false>(p, st);
  if (dtype == F16) return vec ? norm::fwd_any<__half, true>(p, st)
                               : norm::fwd_any<__half, false>(p, st);
  return vec ? norm::fwd_any<float, true>(p, st) : norm::fwd_any<float, false>(p, st);
}

extern "C" int gsq_residual_norm_bwd_workspace(int T, int H, int dtype, int gate_rows,
                                               int64_t* bytes) {
  if (T <= 0 || T > kMaxDim || H <= 0 || dtype < 0 || dtype > 2 || gate_rows < 0 || (gate_rows && T % gate_rows) || !bytes)
    return GSQ_EINVAL;
  *bytes = norm::bwd_plan(T, H, dtype, gate_rows ? gate_rows : 1, gate_rows > 0).ws *
           (int64_t)sizeof(float);
  return GSQ_OK;
}

extern "C" int gsq_residual_norm_bwd(const void* h, int64_t ld_h, const void* y, int64_t ld_y,
                                     const void* w_post, const void* w_pre, const void* gate,
                                     int gate_rows, const float* stats, const void* dh2,
                                     int64_t ld_dh2, const void* dx, int64_t ld_dx, int T, int H,
                                     int dtype, float alpha, float offset, void* dh,
                                     int64_t ld_dh, void* dy, int64_t ld_dy, float* dw_post,
                                     float* dw_pre, float* dgate, float* workspace,
                                     int64_t workspace_bytes, int* err, void* stream) {
  if (T <= 0 || T > kMaxDim || H <= 0 || dtype < 0 || dtype > 2 || !stats || !err) return GSQ_EINVAL;
  const size_t es = dtype_size(dtype);
  if (!norm::row_ok(h, ld_h, H, es) || !norm::row_ok(y, ld_y, H, es) ||
      !norm::row_ok(dh, ld_dh, H, es) || !norm::row_ok(dy, ld_dy, H, es))
    return GSQ_EINVAL;
  if (!lies_on(w_post, es) || !lies_on(w_pre, es) || !lies_on(gate, es) || !lies_on(stats, 4) ||
      !lies_on(dw_post, 4) || !lies_on(dw_pre, 4) || !lies_on(dgate, 4) || !lies_on(err, 4))
    return GSQ_EINVAL;
  if ((gate && (gate_rows <= 0 || T % gate_rows || !dgate)) || (!gate && dgate)) return GSQ_EINVAL;
  if ((dh2 && !norm::row_ok(dh2, ld_dh2, H, es)) || (w_post && !dw_post) || (w_pre && !dw_pre) ||
      (w_pre ? !norm::row_ok(dx, ld_dx, H, es) : dx != nullptr) || (!dh2 && !w_pre))
    return GSQ_EINVAL;
  if (H > norm::kMaxH) return GSQ_ENOTSUP;
  const int groups = gate ? gate_rows : 1;
  const norm::Plan pl = norm::bwd_plan(T, H, dtype, groups, gate != nullptr);
  if (!workspace || (uintptr_t)workspace % 4 || workspace_bytes < pl.ws * (int64_t)sizeof(float))
    return GSQ_EINVAL;
  norm::Bwd p;
  p.in[0] = y; p.in[1] = h; p.in[2] = dx; p.in[3] = dh2;
  p.ld[0] = ld_y; p.ld[1] = ld_h; p.ld[2] = ld_dx; p.ld[3] = ld_dh2;
  p.w_post = w_post; p.w_pre = w_pre; p.gate = gate; p.stats = stats;
  p.T = T; p.H = H; p.per_gate = T / groups;
  p.alpha = alpha; p.offset = offset;
  p.dh = dh; p.ld_dh = ld_dh; p.dy = dy; p.ld_dy = ld_dy;
  p.groups = groups; p.splits = pl.splits; p.slots = pl.slots; p.row_bytes = pl.row_bytes;
  p.err = err;
  p.part_w = workspace;
  p.part_g = !gate ? nullptr
                   : (pl.splits == 1 ? dgate : workspace + (int64_t)pl.teams * 2 * H);
  const bool vec = H % 4 == 0 && norm::row_vec(h, ld_h, es) && norm::row_vec(y, ld_y, es) &&
                   norm::row_vec(w_post, 0, es) && norm::row_vec(w_pre, 0, es) &&
                   norm::row_vec(gate, H, es) && norm::row_vec(dh2, ld_dh2, es) &&
                   norm::row_vec(dx, ld_dx, es) && norm::row_vec(dh, ld_dh, es) &&
                   norm::row_vec(dy, ld_dy, es);
  cudaStream_t st = (cudaStream_t)stream;
  int s;
  if (dtype == BF16) s = vec ? norm::bwd_any<__nv_bfloat16, true>(p, pl, st)
                             : norm::bwd_any<__nv_bfloat16, false>(p, pl, st);
  else if (dtype == F16) s = vec ? norm::bwd_any<__half, true>(p, pl, st)
                                 : norm::bwd_any<__half, false>(p, pl, st);
  else s = vec ? norm::bwd_any<float, true>(p, pl, st) : norm::bwd_any<float, false>(p, pl, st);
  if (s != GSQ_OK) return s;
  const bool gsum = gate && pl.splits > 1;
  const norm::Reduce r0 = {workspace, w_post ? dw_post : nullptr, pl.teams, 0, 2 * (int64_t)H};
  const norm::Reduce r1 = {workspace + H, w_pre ? dw_pre : nullptr, pl.teams, 0, 2 * (int64_t)H};
  const norm::Reduce r2 = {p.part_g, gsum ? dgate : nullptr, pl.splits, pl.splits, H};
  if (w_post || w_pre || gsum) {
    norm::reduce_kernel<<<dim3((H + 31) / 32, 2 + (gsum ? groups : 0)), 1024, 0, st>>>(r0, r1, r2,
                                                                                       H);
    GSQ_CHECK_LAUNCH();
  }
  return GSQ_OK;
}
