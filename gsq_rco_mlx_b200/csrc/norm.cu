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
// Both directions are one pass over their rows, held in registers by a team of threads (a warp
// up to 1024 columns, a block above), so they are bound by the bytes of the rows.
// The column sums of the backward pass: each team adds its rows in registers and writes one
// partial row; a second kernel adds the partials in a fixed order (no atomics: the same inputs
// give the same bits).
#include "dtypes.cuh"

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

struct Bwd {
  const void *h, *y, *w_post, *w_pre, *gate;
  int64_t ld_h, ld_y;
  const float* stats;
  const void *dh2, *dx;  // dh2 may be NULL (zeros), dx NULL without w_pre
  int64_t ld_dh2, ld_dx;
  int T, H, per_gate;
  float alpha, offset;
  void *dh, *dy;
  int64_t ld_dh, ld_dy;
  int groups, splits;  // gate rows, and the parts each one's rows are cut into
  float* part_w;       // [teams][2][H] partials of dw_post, dw_pre
  float* part_g;       // [groups * splits][H] partials of dgate (dgate itself if splits == 1)
};

// Sum over the TPR threads of a row's team. Teams of more than a warp are a whole block, whose
// two staging rows alternate so that one barrier per sum is enough.
template <int TPR>
__device__ __forceinline__ float team_sum(float v, float (*red)[32], int& turn) {
  v = warp_sum(v);
  if (TPR == 32) return v;
  constexpr int NW = TPR / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* r = red[turn & 1];
  ++turn;
  if (lane == 0) r[warp] = v;
  __syncthreads();
  float s = lane < NW ? r[lane] : 0.f;
  return warp_sum(s);
}

template <typename T, bool VEC, int TPR, int NC, bool FP8>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR) fwd_kernel(const __grid_constant__ Fwd p) {
  __shared__ float red[2][32];
  int turn = 0;
  const int t = TPR == 32 ? threadIdx.x & 31 : threadIdx.x;
  const int teams = TPR == 32 ? 8 : 1;
  const int row = blockIdx.x * teams + (TPR == 32 ? threadIdx.x >> 5 : 0);
  if (row >= p.T) return;  // (a whole warp, or a whole block)
  const float inv_H = 1.f / (float)p.H;
  const T* hr = reinterpret_cast<const T*>(p.h) + (int64_t)row * p.ld_h;
  const T* yr = reinterpret_cast<const T*>(p.y) + (int64_t)row * p.ld_y;
  float y[NC][8], h[NC][8];
#pragma unroll
  for (int c = 0; c < NC; ++c) load8<T, VEC>(yr, (c * TPR + t) * 8, p.H, y[c]);
#pragma unroll
  for (int c = 0; c < NC; ++c) load8<T, VEC>(hr, (c * TPR + t) * 8, p.H, h[c]);
  float r1 = 1.f;
  if (p.w_post) {
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) s = fmaf(y[c][j], y[c][j], s);
    r1 = rsqrtf(team_sum<TPR>(s, red, turn) * inv_H + p.eps);
  }
  const T* gr = p.gate ? reinterpret_cast<const T*>(p.gate) + (int64_t)(row / p.per_gate) * p.H
                       : nullptr;
  float s = 0.f;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int col = (c * TPR + t) * 8;
    if (p.w_post) {
      float a[8];
      load8<T, VEC>(reinterpret_cast<const T*>(p.w_post), col, p.H, a);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[c][j] *= r1 * (a[j] + p.offset);
    }
    if (gr) {
      float g[8];
      load8<T, VEC>(gr, col, p.H, g);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[c][j] *= g[j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      h[c][j] = fmaf(p.alpha, y[c][j], h[c][j]);
      s = fmaf(h[c][j], h[c][j], s);
    }
    if (p.h_out)
      store8<T, VEC>(reinterpret_cast<T*>(p.h_out) + (int64_t)row * p.ld_ho, col, p.H, h[c]);
  }
  float r2 = 1.f;
  if (p.w_pre) {
    r2 = rsqrtf(team_sum<TPR>(s, red, turn) * inv_H + p.eps);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int col = (c * TPR + t) * 8;
      float b[8];
      load8<T, VEC>(reinterpret_cast<const T*>(p.w_pre), col, p.H, b);
#pragma unroll
      for (int j = 0; j < 8; ++j) h[c][j] *= r2 * (b[j] + p.offset);
      if (!FP8) {
        store8<T, VEC>(reinterpret_cast<T*>(p.x) + (int64_t)row * p.ld_x, col, p.H, h[c]);
      } else {
        // a 128-column block is the eight columns of each of 16 neighbouring lanes
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (col + j >= p.H) h[c][j] = 0.f;
        float m = amax8(h[c]);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
        m = max_nan(m, kFp8AmaxMin);
        if (col < p.H) {
          if ((t & 15) == 0)
            p.scales[(int64_t)(col / kFp8Block) * p.ld_s + row] = __fdiv_rn(m, kFp8Max);
          *reinterpret_cast<uint2*>(p.codes + (int64_t)row * p.ld_c + col) =
              encode8(h[c], __fdiv_rn(kFp8Max, m));
        }
      }
    }
  }
  if (t == 0) {
    p.stats[row] = r1;
    p.stats[p.T + row] = r2;
  }
}

template <typename T, bool VEC, int TPR, int NC>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR) bwd_kernel(const __grid_constant__ Bwd p) {
  __shared__ float red[2][32];
  int turn = 0;
  const int t = TPR == 32 ? threadIdx.x & 31 : threadIdx.x;
  const int per_block = TPR == 32 ? 8 : 1;
  const int team = blockIdx.x * per_block + (TPR == 32 ? threadIdx.x >> 5 : 0);
  const int teams = gridDim.x * per_block;
  const float inv_H = 1.f / (float)p.H;
  float sw_post[NC][8], sw_pre[NC][8];
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int j = 0; j < 8; ++j) sw_post[c][j] = sw_pre[c][j] = 0.f;
  for (int64_t item = team; item < (int64_t)p.groups * p.splits; item += teams) {
    const int g = (int)(item / p.splits), part = (int)(item - (int64_t)g * p.splits);
    const int lo = (int)((int64_t)p.per_gate * part / p.splits) + g * p.per_gate;
    const int hi = (int)((int64_t)p.per_gate * (part + 1) / p.splits) + g * p.per_gate;
    const T* gr = p.gate ? reinterpret_cast<const T*>(p.gate) + (int64_t)g * p.H : nullptr;
    float sg[NC][8];
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) sg[c][j] = 0.f;
    for (int row = lo; row < hi; ++row) {
      float y[NC][8], h[NC][8], u[NC][8], d[NC][8];
      const T* yr = reinterpret_cast<const T*>(p.y) + (int64_t)row * p.ld_y;
      const T* hr = reinterpret_cast<const T*>(p.h) + (int64_t)row * p.ld_h;
#pragma unroll
      for (int c = 0; c < NC; ++c) load8<T, VEC>(yr, (c * TPR + t) * 8, p.H, y[c]);
#pragma unroll
      for (int c = 0; c < NC; ++c) load8<T, VEC>(hr, (c * TPR + t) * 8, p.H, h[c]);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        if (p.dh2)
          load8<T, VEC>(reinterpret_cast<const T*>(p.dh2) + (int64_t)row * p.ld_dh2,
                        (c * TPR + t) * 8, p.H, d[c]);
        else
#pragma unroll
          for (int j = 0; j < 8; ++j) d[c][j] = 0.f;
        if (p.w_pre)
          load8<T, VEC>(reinterpret_cast<const T*>(p.dx) + (int64_t)row * p.ld_dx,
                        (c * TPR + t) * 8, p.H, u[c]);
      }
      const float r1 = p.w_post ? p.stats[row] : 1.f, r2 = p.w_pre ? p.stats[p.T + row] : 1.f;
      float s = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int col = (c * TPR + t) * 8;
        float a[8], gv[8];
        if (p.w_post) load8<T, VEC>(reinterpret_cast<const T*>(p.w_post), col, p.H, a);
        if (gr) load8<T, VEC>(gr, col, p.H, gv);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float n = y[c][j] * r1;
          if (p.w_post) n *= a[j] + p.offset;
          if (gr) n *= gv[j];
          h[c][j] = fmaf(p.alpha, n, h[c][j]) * r2;  // h' r2
        }
        if (p.w_pre) {
          float b[8];
          load8<T, VEC>(reinterpret_cast<const T*>(p.w_pre), col, p.H, b);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            sw_pre[c][j] = fmaf(u[c][j], h[c][j], sw_pre[c][j]);
            u[c][j] *= b[j] + p.offset;
            s = fmaf(u[c][j], h[c][j], s);
          }
        }
      }
      if (p.w_pre) {
        const float mu = team_sum<TPR>(s, red, turn) * inv_H;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int j = 0; j < 8; ++j) d[c][j] = fmaf(r2, u[c][j] - h[c][j] * mu, d[c][j]);
      }
      float s2 = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int col = (c * TPR + t) * 8;
        store8<T, VEC>(reinterpret_cast<T*>(p.dh) + (int64_t)row * p.ld_dh, col, p.H, d[c]);
        float a[8], gv[8];
        if (p.w_post) load8<T, VEC>(reinterpret_cast<const T*>(p.w_post), col, p.H, a);
        if (gr) load8<T, VEC>(gr, col, p.H, gv);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float yn = y[c][j] * r1, ad = p.alpha * d[c][j];
          const float aj = p.w_post ? a[j] + p.offset : 1.f;
          sg[c][j] = fmaf(ad, yn * aj, sg[c][j]);
          const float m = gr ? ad * gv[j] : ad;
          sw_post[c][j] = fmaf(m, yn, sw_post[c][j]);
          u[c][j] = m * aj;   // v
          y[c][j] = yn;
          s2 = fmaf(u[c][j], yn, s2);
        }
      }
      const float mv = p.w_post ? team_sum<TPR>(s2, red, turn) * inv_H : 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
#pragma unroll
        for (int j = 0; j < 8; ++j) u[c][j] = r1 * (u[c][j] - y[c][j] * mv);
        store8<T, VEC>(reinterpret_cast<T*>(p.dy) + (int64_t)row * p.ld_dy, (c * TPR + t) * 8, p.H,
                       u[c]);
      }
    }
    if (p.part_g) {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int col = (c * TPR + t) * 8;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (col + j < p.H) p.part_g[item * p.H + col + j] = sg[c][j];
      }
    }
  }
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int col = (c * TPR + t) * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (col + j < p.H) {
        p.part_w[((int64_t)team * 2) * p.H + col + j] = sw_post[c][j];
        p.part_w[((int64_t)team * 2 + 1) * p.H + col + j] = sw_pre[c][j];
      }
  }
}

// out[o][c] = sum over i < n of part[(o outer + i) stride + c]: a block takes 32 columns of one
// output row, eight threads a column; the order of the sums does not depend on the launch.
struct Reduce {
  const float* part;
  float* out;
  int n;
  int64_t outer, stride;
};

__global__ void __launch_bounds__(256)
reduce_kernel(Reduce r0, Reduce r1, Reduce r2, int H, int64_t rows2) {
  __shared__ float s[8][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + lane;
  const int64_t o = blockIdx.y < 2 ? 0 : blockIdx.y - 2;
  const Reduce& r = blockIdx.y == 0 ? r0 : (blockIdx.y == 1 ? r1 : r2);
  if (!r.out) return;
  float a = 0.f;
  if (col < H)
    for (int i = w; i < r.n; i += 8) a += r.part[(o * r.outer + i) * r.stride + col];
  s[w][lane] = a;
  __syncthreads();
  if (w == 0 && col < H) {
#pragma unroll
    for (int i = 1; i < 8; ++i) a += s[i][lane];
    r.out[o * H + col] = a;
  }
}

constexpr int kMaxH = 32768;

template <typename T, bool VEC, int TPR, int NC>
static int fwd_launch(const Fwd& p, cudaStream_t st) {
  const int per = TPR == 32 ? 8 : 1, threads = TPR == 32 ? 256 : TPR;
  const unsigned g = (unsigned)((p.T + per - 1) / per);
  if (p.codes) fwd_kernel<T, VEC, TPR, NC, true><<<g, threads, 0, st>>>(p);
  else fwd_kernel<T, VEC, TPR, NC, false><<<g, threads, 0, st>>>(p);
  GSQ_CHECK_LAUNCH();
  return GSQ_OK;
}

template <typename T, bool VEC>
static int fwd_any(const Fwd& p, cudaStream_t st) {
  const int v = (p.H + 7) / 8;
  if (v <= 32) return fwd_launch<T, VEC, 32, 1>(p, st);
  if (v <= 64) return fwd_launch<T, VEC, 32, 2>(p, st);
  if (v <= 128) return fwd_launch<T, VEC, 32, 4>(p, st);
  if (v <= 256) return fwd_launch<T, VEC, 64, 4>(p, st);
  if (v <= 512) return fwd_launch<T, VEC, 128, 4>(p, st);
  if (v <= 1024) return fwd_launch<T, VEC, 256, 4>(p, st);
  if (v <= 2048) return fwd_launch<T, VEC, 512, 4>(p, st);
  return fwd_launch<T, VEC, 1024, 4>(p, st);
}

// Teams of the backward pass, and the parts each gate row's rows are cut into: as many teams as
// stay resident, and parts so that every team has rows.
struct Plan {
  int blocks, teams, splits;
  int64_t ws;  // floats of workspace
};

static Plan bwd_plan(int T, int H, int groups, bool gate) {
  Plan pl;
  const int v = (H + 7) / 8, per = v <= 128 ? 8 : 1;
  const int most = num_sms() * (v <= 128 ? 1 : (v <= 256 ? 6 : (v <= 512 ? 3 : (v <= 1024 ? 2 : 1))));
  int64_t blocks = ((int64_t)T + per - 1) / per;
  if (blocks > most) blocks = most;
  pl.blocks = (int)blocks;
  pl.teams = pl.blocks * per;
  const int rows = T / groups;
  int s = (pl.teams + groups - 1) / groups;
  if (s > rows) s = rows;
  pl.splits = s;
  pl.ws = (int64_t)pl.teams * 2 * H + (gate && s > 1 ? (int64_t)groups * s * H : 0);
  return pl;
}

template <typename T, bool VEC>
static int bwd_any(const Bwd& p, const Plan& pl, cudaStream_t st) {
  const int v = (p.H + 7) / 8;
  const unsigned g = (unsigned)pl.blocks;
  if (v <= 32) bwd_kernel<T, VEC, 32, 1><<<g, 256, 0, st>>>(p);
  else if (v <= 64) bwd_kernel<T, VEC, 32, 2><<<g, 256, 0, st>>>(p);
  else if (v <= 128) bwd_kernel<T, VEC, 32, 4><<<g, 256, 0, st>>>(p);
  else if (v <= 256) bwd_kernel<T, VEC, 128, 2><<<g, 128, 0, st>>>(p);
  else if (v <= 512) bwd_kernel<T, VEC, 256, 2><<<g, 256, 0, st>>>(p);
  else if (v <= 1024) bwd_kernel<T, VEC, 512, 2><<<g, 512, 0, st>>>(p);
  else if (v <= 2048) bwd_kernel<T, VEC, 1024, 2><<<g, 1024, 0, st>>>(p);
  else bwd_kernel<T, VEC, 1024, 4><<<g, 1024, 0, st>>>(p);
  GSQ_CHECK_LAUNCH();
  return GSQ_OK;
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
  if (T <= 0 || H <= 0 || dtype < 0 || dtype > 2 || !stats) return GSQ_EINVAL;
  const size_t es = dtype_size(dtype);
  if (!norm::row_ok(h, ld_h, H, es) || !norm::row_ok(y, ld_y, H, es)) return GSQ_EINVAL;
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
  const bool vec = norm::row_vec(h, ld_h, es) && norm::row_vec(y, ld_y, es) &&
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

extern "C" int gsq_residual_norm_bwd_workspace(int T, int H, int gate_rows, int64_t* bytes) {
  if (T <= 0 || H <= 0 || gate_rows < 0 || (gate_rows && T % gate_rows) || !bytes)
    return GSQ_EINVAL;
  *bytes = norm::bwd_plan(T, H, gate_rows ? gate_rows : 1, gate_rows > 0).ws *
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
                                     int64_t workspace_bytes, void* stream) {
  if (T <= 0 || H <= 0 || dtype < 0 || dtype > 2 || !stats) return GSQ_EINVAL;
  const size_t es = dtype_size(dtype);
  if (!norm::row_ok(h, ld_h, H, es) || !norm::row_ok(y, ld_y, H, es) ||
      !norm::row_ok(dh, ld_dh, H, es) || !norm::row_ok(dy, ld_dy, H, es))
    return GSQ_EINVAL;
  if ((gate && (gate_rows <= 0 || T % gate_rows || !dgate)) || (!gate && dgate)) return GSQ_EINVAL;
  if ((dh2 && !norm::row_ok(dh2, ld_dh2, H, es)) || (w_post && !dw_post) || (w_pre && !dw_pre) ||
      (w_pre ? !norm::row_ok(dx, ld_dx, H, es) : dx != nullptr) || (!dh2 && !w_pre))
    return GSQ_EINVAL;
  if (H > norm::kMaxH) return GSQ_ENOTSUP;
  const int groups = gate ? gate_rows : 1;
  const norm::Plan pl = norm::bwd_plan(T, H, groups, gate != nullptr);
  if (!workspace || (uintptr_t)workspace % 4 || workspace_bytes < pl.ws * (int64_t)sizeof(float))
    return GSQ_EINVAL;
  norm::Bwd p;
  p.h = h; p.y = y; p.w_post = w_post; p.w_pre = w_pre; p.gate = gate;
  p.ld_h = ld_h; p.ld_y = ld_y; p.stats = stats;
  p.dh2 = dh2; p.ld_dh2 = ld_dh2; p.dx = dx; p.ld_dx = ld_dx;
  p.T = T; p.H = H; p.per_gate = T / groups;
  p.alpha = alpha; p.offset = offset;
  p.dh = dh; p.ld_dh = ld_dh; p.dy = dy; p.ld_dy = ld_dy;
  p.groups = groups; p.splits = pl.splits;
  p.part_w = workspace;
  p.part_g = !gate ? nullptr
                   : (pl.splits == 1 ? dgate : workspace + (int64_t)pl.teams * 2 * H);
  const bool vec = norm::row_vec(h, ld_h, es) && norm::row_vec(y, ld_y, es) &&
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
    norm::reduce_kernel<<<dim3((H + 31) / 32, 2 + (gsum ? groups : 0)), 256, 0, st>>>(r0, r1, r2,
                                                                                      H, groups);
    GSQ_CHECK_LAUNCH();
  }
  return GSQ_OK;
}
