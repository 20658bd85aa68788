// Rotary positions of q and k: every pair (a, b) of a head's rotated part turns by t = p w_j,
//   (a, b) -> f (a cos t - b sin t, a sin t + b cos t)
// with p the token's position, w_j the pair's frequency and f a factor of the plan; its
// vector-Jacobian product is the same with -t. The rest of the head passes through.
//
// Far positions: t is held as turns, p (w_j / 2 pi), in 64 bits; the whole turns are taken off
// there, and sincospif sees the remainder in [-1/2, 1/2] turns. So the angle is off by the float32
// rounding of that remainder (2^-25 pi, 1e-7 radians) and by 2^-52 of the whole angle (the rounding
// of the stored frequency and of the product): 1e-8 radians at p w_j = 5e7, 5e-7 at 2^31.
//
// Bound by the bytes of q and k, read once and written once. A thread owns one vector of pairs
// of one token in up to four heads, so the 64-bit angles and the sines are computed once for
// several heads, while their loads are in flight: no table of positions is read. 16384 x 16 heads
// of 64 in bf16: 17 us, 3.9 TB/s; 8191 x 40 heads of 128 in float16: 33 us, 5.1 TB/s.
#include "dtypes.cuh"

namespace gsq {
namespace rope {

struct Side {
  const void* in;
  void* out;
  int64_t in_t, in_h, out_t, out_h;  // element strides of tokens and heads
  int heads;
};

struct Args {
  Side q, k;
  const void* pos;
  int pos64;
  const double* turns;  // [rot / 2] w_j / 2 pi
  float factor, sign;
  int64_t T;
  int hd, rot;
  int lanes;   // vectors of a head
  int chunks;  // thread groups a token's heads are dealt to
  int tokens;  // tokens per block
};

template <int N>
struct Bytes;
template <> struct Bytes<2> { typedef uint16_t type; };
template <> struct Bytes<4> { typedef uint32_t type; };
template <> struct Bytes<8> { typedef uint2 type; };
template <> struct Bytes<16> { typedef uint4 type; };

template <typename T, int V>
struct __align__(sizeof(T) * V) Vec {
  T e[V];
};

template <typename T, int V>
__device__ __forceinline__ Vec<T, V> ld(const T* p) {
  typedef typename Bytes<sizeof(T) * V>::type B;
  Vec<T, V> v;
  *reinterpret_cast<B*>(&v) = *reinterpret_cast<const B*>(p);
  return v;
}

template <typename T, int V>
__device__ __forceinline__ void st(T* p, const Vec<T, V>& v) {
  typedef typename Bytes<sizeof(T) * V>::type B;
  *reinterpret_cast<B*>(p) = *reinterpret_cast<const B*>(&v);
}

template <typename T>
__device__ __forceinline__ const T* side_in(const Args& p, int h, int64_t t) {
  return h < p.q.heads
             ? reinterpret_cast<const T*>(p.q.in) + t * p.q.in_t + h * p.q.in_h
             : reinterpret_cast<const T*>(p.k.in) + t * p.k.in_t + (h - p.q.heads) * p.k.in_h;
}

template <typename T>
__device__ __forceinline__ T* side_out(const Args& p, int h, int64_t t) {
  return h < p.q.heads
             ? reinterpret_cast<T*>(p.q.out) + t * p.q.out_t + h * p.q.out_h
             : reinterpret_cast<T*>(p.k.out) + t * p.k.out_t + (h - p.q.heads) * p.k.out_h;
}

constexpr int kBatch = 4;  // heads whose loads are in flight before the first is turned

// V elements a load. Halves: lane v < rot / 2 / V holds elements v V.. and their partners
// rot / 2 further. Pairs (INTER): lane v < rot / V holds V / 2 pairs (V = 1: a pair, two
// elements). Lanes behind them copy the rest of the head.
template <typename T, int V, bool INTER>
__global__ void __launch_bounds__(256) rope_kernel(const __grid_constant__ Args p) {
  constexpr int NP = INTER ? (V == 1 ? 1 : V / 2) : V;  // pairs of a lane
  const int per = p.lanes * p.chunks;
  const int rot_lanes = INTER ? p.rot / (V == 1 ? 2 : V) : p.rot / 2 / V;
  const int heads = p.q.heads + p.k.heads;
  for (int e = threadIdx.x; e < per * p.tokens; e += blockDim.x) {
    const int tk = e / per, i = e - tk * per;
    const int64_t t = (int64_t)blockIdx.x * p.tokens + tk;
    if (t >= p.T) return;
    const int c = i / p.lanes, v = i - c * p.lanes;
    const bool turn = v < rot_lanes;
    const int o1 = turn ? (INTER ? v * (V == 1 ? 2 : V) : v * V)
                        : p.rot + (v - rot_lanes) * V;
    const int d = INTER ? 1 : p.rot / 2;  // where the partner of an element lies
    constexpr bool kTwo = !INTER || V == 1;
    Vec<T, V> x[kBatch], y[kTwo ? kBatch : 1];
    auto load = [&](int h0) {
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int h = h0 + b * p.chunks;
        if (h < heads) {
          const T* in = side_in<T>(p, h, t) + o1;
          x[b] = ld<T, V>(in);
          if (kTwo && turn) y[kTwo ? b : 0] = ld<T, V>(in + d);
        }
      }
    };
    load(c);   // the first heads are on their way while the angles are worked out
    float cs[NP], sn[NP];
    if (turn) {
      const double pos = p.pos64 ? (double)reinterpret_cast<const int64_t*>(p.pos)[t]
                                 : (double)reinterpret_cast<const int32_t*>(p.pos)[t];
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        const double a = pos * p.turns[v * NP + j];
        const float r = (float)(2.0 * (a - rint(a)));
        float s, co;
        sincospif(r, &s, &co);
        cs[j] = co * p.factor;
        sn[j] = s * (p.factor * p.sign);
      }
    }
    for (int h0 = c; h0 < heads; h0 += kBatch * p.chunks) {
      if (h0 != c) load(h0);
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int h = h0 + b * p.chunks;
        if (h < heads) {
          T* out = side_out<T>(p, h, t) + o1;
          if (turn) {
            if (!kTwo) {
#pragma unroll
              for (int j = 0; j < NP; ++j) {
                const float u = to_f32(x[b].e[2 * j]), w = to_f32(x[b].e[V > 1 ? 2 * j + 1 : 0]);
                x[b].e[2 * j] = from_f32<T>(u * cs[j] - w * sn[j]);
                x[b].e[V > 1 ? 2 * j + 1 : 0] = from_f32<T>(u * sn[j] + w * cs[j]);
              }
            } else {
              Vec<T, V>& z = y[kTwo ? b : 0];
#pragma unroll
              for (int j = 0; j < NP; ++j) {
                const float u = to_f32(x[b].e[j]), w = to_f32(z.e[j]);
                x[b].e[j] = from_f32<T>(u * cs[j] - w * sn[j]);
                z.e[j] = from_f32<T>(u * sn[j] + w * cs[j]);
              }
              st<T, V>(out + d, z);
            }
          }
          st<T, V>(out, x[b]);
        }
      }
    }
  }
}

inline bool fits(const Side& s, size_t es, int V) {
  const size_t b = es * V;
  return s.heads == 0 ||
         ((uintptr_t)s.in % b == 0 && (uintptr_t)s.out % b == 0 && s.in_t % V == 0 &&
          s.in_h % V == 0 && s.out_t % V == 0 && s.out_h % V == 0);
}

template <typename T, bool INTER>
static int launch(Args& p, cudaStream_t st) {
  // the widest vector that divides the head's parts, the strides and the addresses
  int V = 16 / sizeof(T);
  for (; V > 1; V /= 2)
    if (p.hd % V == 0 && p.rot % (INTER ? V : 2 * V) == 0 && fits(p.q, sizeof(T), V) &&
        fits(p.k, sizeof(T), V))
      break;
  const int rot_lanes = INTER ? p.rot / (V == 1 ? 2 : V) : p.rot / 2 / V;
  const bool same = p.q.in == p.q.out && (p.k.heads == 0 || p.k.in == p.k.out);
  p.lanes = rot_lanes + (same ? 0 : (p.hd - p.rot) / V);
  const int heads = p.q.heads + p.k.heads;
  // Heads a thread turns by its angles: four where that leaves 192 threads an SM (16384 x 16 heads
  // of 64 in bf16: 18.0 us, with two 23.1, with one 36.4; 2048: 4.8, 5.0, 6.8), fewer for fewer
  // tokens (1024: 3.7, 3.3, 3.7; 512: 3.6, 3.1, 2.9; 1: 2.9, 2.5, 2.3), unless a token's threads
  // would no longer be one turn of a block (1 x 40 heads of 128: with two 2.9, with one 3.8). Eight
  // in two batches: 19.8 at 16384 x 16, 35.9 for 32.8 at 8191 x 40.
  int walk = kBatch;
  while (walk > 1 && p.T * p.lanes * ((heads + walk - 1) / walk) < (int64_t)num_sms() * 192 &&
         p.lanes * ((heads + walk / 2 - 1) / (walk / 2)) <= 256)
    walk /= 2;
  p.chunks = (heads + walk - 1) / walk;
  const int per = p.lanes * p.chunks;
  p.tokens = per >= 256 ? 1 : 256 / per;
  const int64_t blocks = (p.T + p.tokens - 1) / p.tokens;
  if (blocks > INT32_MAX) return GSQ_EINVAL;
  const int threads = per >= 256 ? 256 : (per * p.tokens + 31) / 32 * 32;
#define GSQ_ROPE(VV) rope_kernel<T, VV, INTER><<<(unsigned)blocks, threads, 0, st>>>(p)
  if (V == 8) {
    if constexpr (sizeof(T) == 2) GSQ_ROPE(8);
  } else if (V == 4) GSQ_ROPE(4);
  else if (V == 2) GSQ_ROPE(2);
  else GSQ_ROPE(1);
#undef GSQ_ROPE
  GSQ_CHECK_LAUNCH();
  return GSQ_OK;
}

}  // namespace rope
}  // namespace gsq

using namespace gsq;

extern "C" int gsq_rope(const void* q, int64_t q_t, int64_t q_h, int nq, const void* k,
                        int64_t k_t, int64_t k_h, int nk, int64_t T, int head_dim,
                        int rotary_dim, int interleaved, int dtype, const void* positions,
                        int positions64, const double* turns, float factor, int inverse,
                        void* q_out, int64_t qo_t, int64_t qo_h, void* k_out, int64_t ko_t,
                        int64_t ko_h, void* stream) {
  if (!q || !q_out || nq <= 0 || nk < 0 || (nk > 0 && (!k || !k_out)) || T <= 0 ||
      head_dim <= 0 || rotary_dim <= 0 || rotary_dim % 2 || rotary_dim > head_dim || dtype < 0 ||
      dtype > 2 || !positions || !turns || (uintptr_t)positions % (positions64 ? 8 : 4) ||
      (uintptr_t)turns % 8 || nq > 65536 || nk > 65536 || head_dim > 65536)
    return GSQ_EINVAL;
  const size_t es = dtype_size(dtype);
  if ((uintptr_t)q % es || (uintptr_t)q_out % es || (nk && ((uintptr_t)k % es || (uintptr_t)k_out % es)))
    return GSQ_EINVAL;
  rope::Args p;
  p.q = {q, q_out, q_t, q_h, qo_t, qo_h, nq};
  p.k = {k, k_out, k_t, k_h, ko_t, ko_h, nk};
  p.pos = positions;
  p.pos64 = positions64;
  p.turns = turns;
  p.factor = factor;
  p.sign = inverse ? -1.f : 1.f;
  p.T = T;
  p.hd = head_dim;
  p.rot = rotary_dim;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == BF16) return interleaved ? rope::launch<__nv_bfloat16, true>(p, st)
                                        : rope::launch<__nv_bfloat16, false>(p, st);
  if (dtype == F16) return interleaved ? rope::launch<__half, true>(p, st)
                                       : rope::launch<__half, false>(p, st);
  return interleaved ? rope::launch<float, true>(p, st) : rope::launch<float, false>(p, st);
}
