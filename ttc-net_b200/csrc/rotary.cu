// Rotary positions: pair p of a head's first 2 half values turns by angle = position * inv_freq[p],
//   (a, b) -> m (a cos - b sin, a sin + b cos),
// pairs (p, p + half) or, interleaved, (2p, 2p + 1); values behind 2 half are copied.  The backward
// is the turn by -angle with the same factor m.
//
// The angle is formed and reduced to [-pi, pi] in 64 bits: at position 10^6 one 32-bit rounding of
// it is 0.03 rad.  A CTA takes a few tokens (256 / half of them, so that a thread has about one pair), computes their
// cosines and sines once into shared memory and streams the heads of q and k past them.  Bound by memory,
// each value is read and written once: 335 MB (4 x 4096 tokens, 32 + 8 heads of 128, bf16) take 60 us, 5.5 TB/s or
// 0.85 of the copy rate; interleaved 68 us, the same bytes in fp32 58 us (half the angles).  What it took against
// 67, 77 and 60 us of the first form: loads in flight during the sines, several heads loaded before one is stored, and
// a table that is read without bank conflicts.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cstdio>

#include "lqr_common.cuh"
#include "ttc_b200.h"

namespace ttc {
int set_error(int code, const char* msg);
}

namespace {

using ttc::ldf;
using ttc::stf;

constexpr int kThreads = 256;
constexpr int kMaxTokens = 16;

struct Rot {
  const void* x[2];  // q, k (k may be null with 0 heads)
  int64_t sb[2], st[2], sh[2];
  void* y[2];  // [B, T, H, D] contiguous
  int H[2];
  const void* pos;
  int64_t pb, pt;
  int pos64;
  const double* inv_freq;
  int64_t B, T;
  int D, half, interleaved;
  double sign;
  float mag;
  int tokens;    // of a CTA
  int heads;     // of a CTA (of q's and k's together)
};

// V values as they lie in memory, and as floats.
template <typename T, int V>
struct Raw;
template <typename T>
struct Raw<T, 1> {
  T x;
  __device__ __forceinline__ void load(const T* p) { x = *p; }
  __device__ __forceinline__ void store(T* p) const { *p = x; }
  __device__ __forceinline__ void get(float (&v)[1]) const { v[0] = ldf(&x); }
  __device__ __forceinline__ void set(const float (&v)[1]) { stf(&x, v[0]); }
};
template <>
struct Raw<float, 4> {
  float4 x;
  __device__ __forceinline__ void load(const float* p) { x = *reinterpret_cast<const float4*>(p); }
  __device__ __forceinline__ void store(float* p) const { *reinterpret_cast<float4*>(p) = x; }
  __device__ __forceinline__ void get(float (&v)[4]) const { v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w; }
  __device__ __forceinline__ void set(const float (&v)[4]) { x = make_float4(v[0], v[1], v[2], v[3]); }
};
template <>
struct Raw<__nv_bfloat16, 8> {
  uint4 x;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { x = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void store(__nv_bfloat16* p) const { *reinterpret_cast<uint4*>(p) = x; }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(u[i] << 16);
      v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  }
  __device__ __forceinline__ void set(const float (&v)[8]) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      u[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    x = make_uint4(u[0], u[1], u[2], u[3]);
  }
};

// A thread's share: one unit of one token, in every `step`-th head.
template <typename T, int V, int HEADS, bool ONE>
struct Share {
  static constexpr int W = V == 1 ? 1 : ONE ? V / 2 : V;  // pairs of a unit
  int at, ia, ib;  // place in the table of cosines and sines, < 0 for a copied vector; a pair's vectors
  int64_t off0, off1;   // of the token in q and k
  int64_t tok;
  Raw<T, V> a[HEADS], b[HEADS];

  __device__ __forceinline__ const T* src(const Rot& P, int h) const {
    return h < P.H[0] ? static_cast<const T*>(P.x[0]) + (off0 + h * P.sh[0])
                      : static_cast<const T*>(P.x[1]) + (off1 + (h - P.H[0]) * P.sh[1]);
  }
  __device__ __forceinline__ T* dst(const Rot& P, int h) const {
    return h < P.H[0] ? static_cast<T*>(P.y[0]) + (tok * P.H[0] + h) * P.D
                      : static_cast<T*>(P.y[1]) + (tok * P.H[1] + h - P.H[0]) * P.D;
  }
  __device__ __forceinline__ void set(const Rot& P, int64_t tok0, int x, int units, int turn) {
    const int t = x / units, u = x - t * units;
    tok = tok0 + t;
    const int64_t n = tok / P.T;
    off0 = n * P.sb[0] + (tok - n * P.T) * P.st[0];
    off1 = n * P.sb[1] + (tok - n * P.T) * P.st[1];
    at = u < turn ? t * turn + u : -1;
    ib = 0;
    if (u >= turn) {
      ia = 2 * P.half + (u - turn) * V;
    } else if (ONE) {
      ia = u * V;
    } else {
      ia = P.interleaved ? 2 * u : u * V, ib = P.interleaved ? 2 * u + 1 : u * V + P.half;
    }
  }
  // HEADS heads are loaded before the first of them is stored: a store may alias a later load for all that the
  // compiler knows.
  __device__ __forceinline__ void load(const Rot& P, int h, int end, int step) {
#pragma unroll
    for (int x = 0; x < HEADS; ++x)
      if (h + x * step < end) {
        const T* const from = src(P, h + x * step);
        a[x].load(from + ia);
        if (!ONE && at >= 0) b[x].load(from + ib);
      }
  }
  __device__ __forceinline__ void turn_store(const Rot& P, const float2* cs, int plane, int h, int end, int step) {
    float2 w[W];
    if (at >= 0) {
      if constexpr (W == 1) {
        w[0] = cs[at];
      } else {
#pragma unroll
        for (int i = 0; i < W; i += 2) {
          const float4 c = reinterpret_cast<const float4*>(cs)[i / 2 * plane + at];
          w[i] = make_float2(c.x, c.y);
          w[i + 1] = make_float2(c.z, c.w);
        }
      }
    }
#pragma unroll
    for (int x = 0; x < HEADS; ++x)
      if (h + x * step < end) {
        T* const to = dst(P, h + x * step);
        if (at >= 0) {
          float p[V];
          a[x].get(p);
          if constexpr (!ONE) {
            float q[V];
            b[x].get(q);
#pragma unroll
            for (int i = 0; i < V; ++i) {
              const float m = p[i], n = q[i];
              p[i] = fmaf(m, w[i].x, -n * w[i].y);
              q[i] = fmaf(m, w[i].y, n * w[i].x);
            }
            b[x].set(q);
            b[x].store(to + ib);
          } else {
#pragma unroll
            for (int i = 0; i < W; ++i) {
              const float m = p[2 * i], n = p[2 * i + 1];
              p[2 * i] = fmaf(m, w[i].x, -n * w[i].y);
              p[2 * i + 1] = fmaf(m, w[i].y, n * w[i].x);
            }
          }
          a[x].set(p);
        }
        a[x].store(to + ia);
      }
  }
};

// Units of a head: `half / V` (pairs of vectors) or, where a vector holds both values of its pairs (ONE: interleaved,
// V > 1), `2 half / V`, then the vectors that are copied.  The table holds two neighbouring pairs of a unit in 16 bytes,
// the units' next to each other (`plane` of them), so that a warp's reads meet no bank twice.
template <typename T, int V, bool ONE>
__global__ void __launch_bounds__(kThreads, 5) rotary_kernel(const __grid_constant__ Rot P) {
  constexpr int HEADS = V == 1 || ONE ? 4 : 2;  // two vectors a head, or one
  extern __shared__ float4 table[];
  float2* const cs = reinterpret_cast<float2*>(table);
  const int64_t tok0 = static_cast<int64_t>(blockIdx.x) * P.tokens;
  const int ntok = static_cast<int>(min(static_cast<int64_t>(P.tokens), P.B * P.T - tok0));
  const int turn = ONE ? 2 * P.half / V : P.half / V, plane = ntok * turn;
  const int units = turn + (P.D - 2 * P.half) / V;
  // thread -> (token, unit), groups of such threads share the heads; the first heads' loads are in flight while the
  // cosines and sines are computed
  const int work = ntok * units, lanes = min(work, kThreads), step = kThreads / lanes;
  const int group = threadIdx.x / lanes, h0 = blockIdx.y * P.heads + group;
  const int end = group < step ? min(static_cast<int>(blockIdx.y + 1) * P.heads, P.H[0] + P.H[1]) : 0;
  int x = threadIdx.x % lanes;
  using My = Share<T, V, HEADS, ONE>;
  My my;
  my.set(P, tok0, x, units, turn);
  my.load(P, h0, end, step);
  for (int i = threadIdx.x; i < ntok * P.half; i += kThreads) {
    const int t = i / P.half, p = i - t * P.half;
    const int64_t tok = tok0 + t, n = tok / P.T, off = n * P.pb + (tok - n * P.T) * P.pt;
    const double pos = P.pos64 ? static_cast<double>(static_cast<const int64_t*>(P.pos)[off])
                               : static_cast<double>(static_cast<const int*>(P.pos)[off]);
    const double angle = P.sign * pos * P.inv_freq[p];
    const double turns = rint(angle * 0.15915494309189535);  // 1 / (2 pi)
    // 2 pi as a sum of two doubles, so that the reduction keeps its digits for many turns
    const double r = fma(-turns, 2.4492935982947064e-16, fma(-turns, 6.283185307179586, angle));
    const float rh = static_cast<float>(r), rl = static_cast<float>(r - static_cast<double>(rh));
    float s, c;
    sincosf(rh, &s, &c);
    const int u = p / My::W, y = p - u * My::W;
    cs[My::W == 1 ? i : (y / 2 * plane + t * turn + u) * 2 + (y & 1)] =
        make_float2(P.mag * fmaf(-s, rl, c), P.mag * fmaf(c, rl, s));
  }
  __syncthreads();
#pragma unroll 1
  while (true) {
#pragma unroll 1
    for (int h = h0; h < end;) {
      my.turn_store(P, cs, plane, h, end, step);
      h += HEADS * step;
      my.load(P, h, end, step);
    }
    x += lanes;
    if (x >= work) break;
    my.set(P, tok0, x, units, turn);
    my.load(P, h0, end, step);
  }
}

int fail(int code, const char* msg) { return ttc::set_error(code, msg); }

template <typename T>
int run(Rot P, cudaStream_t st) {
  constexpr int VT = 16 / sizeof(T);
  bool vec = P.D % VT == 0 && (2 * P.half) % VT == 0 && (P.interleaved || P.half % VT == 0);
  for (int i = 0; i < 2; ++i) {
    if (P.H[i] == 0) continue;
    vec = vec && ((reinterpret_cast<uintptr_t>(P.x[i]) | reinterpret_cast<uintptr_t>(P.y[i])) & 15u) == 0 &&
          P.sb[i] % VT == 0 && P.st[i] % VT == 0 && P.sh[i] % VT == 0;
  }
  const int64_t total = P.B * P.T;
  P.tokens = std::max(1, std::min(kMaxTokens, kThreads / std::max(1, P.half)));
  const int all = P.H[0] + P.H[1];
  P.heads = all;
  // few tokens: fewer of them and of the heads for each CTA
  while (P.tokens > 1 && (total + P.tokens - 1) / P.tokens < 296) P.tokens = (P.tokens + 1) / 2;
  const int64_t ctas = (total + P.tokens - 1) / P.tokens;
  if (ctas < 296) P.heads = std::max<int64_t>(4, (all * ctas + 295) / 296);
  const dim3 grid(static_cast<unsigned>(ctas), (all + P.heads - 1) / P.heads);
  const size_t smem = static_cast<size_t>(P.tokens) * P.half * sizeof(float2);
  if (vec && P.interleaved)
    rotary_kernel<T, VT, true><<<grid, kThreads, smem, st>>>(P);
  else if (vec)
    rotary_kernel<T, VT, false><<<grid, kThreads, smem, st>>>(P);
  else
    rotary_kernel<T, 1, false><<<grid, kThreads, smem, st>>>(P);
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return TTC_OK;
  char buf[256];
  snprintf(buf, sizeof(buf), "rotary_kernel launch: %s", cudaGetErrorString(e));
  return fail(TTC_ERR_CUDA, buf);
}

}  // namespace

extern "C" int ttc_rotary(const void* q, const int64_t* q_strides, int Hq, const void* k, const int64_t* k_strides, int Hk,
                          const void* positions, const int64_t* pos_strides, int pos64, const double* inv_freq,
                          int64_t B, int64_t T, int D, int half, int interleaved, int inverse, float magnitude, int dtype,
                          void* q_out, void* k_out, void* stream) {
  if (B < 0 || T < 0 || B > 0x7fffffffLL || T > 0x7fffffffLL || B * T > 0x7fffffffLL)
    return fail(TTC_ERR_INVALID, "rotary: at most 2^31 - 1 tokens");
  if (Hq < 1 || Hk < 0 || Hq > 65535 || Hk > 65535) return fail(TTC_ERR_INVALID, "rotary: bad number of heads");
  if (D < 1 || D > 512 || half < 0 || 2 * half > D)
    return fail(TTC_ERR_UNSUPPORTED, "rotary: head dim must be in [1, 512], the rotated part at most that");
  if (dtype != TTC_DTYPE_F32 && dtype != TTC_DTYPE_BF16)
    return fail(TTC_ERR_INVALID, "rotary: dtype must be TTC_DTYPE_F32 or TTC_DTYPE_BF16");
  if (B * T == 0) return TTC_OK;
  if (!q || !q_strides || !q_out || (Hk > 0 && (!k || !k_strides || !k_out)) || !positions || !pos_strides ||
      (half > 0 && !inv_freq))
    return fail(TTC_ERR_INVALID, "rotary: null pointer");
  Rot P{};
  P.x[0] = q, P.y[0] = q_out, P.H[0] = Hq, P.sb[0] = q_strides[0], P.st[0] = q_strides[1], P.sh[0] = q_strides[2];
  P.H[1] = Hk;
  if (Hk > 0) P.x[1] = k, P.y[1] = k_out, P.sb[1] = k_strides[0], P.st[1] = k_strides[1], P.sh[1] = k_strides[2];
  P.pos = positions, P.pb = pos_strides[0], P.pt = pos_strides[1], P.pos64 = pos64;
  P.inv_freq = inv_freq, P.B = B, P.T = T, P.D = D, P.half = half, P.interleaved = interleaved;
  P.sign = inverse ? -1.0 : 1.0, P.mag = magnitude;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == TTC_DTYPE_F32 ? run<float>(P, st) : run<__nv_bfloat16>(P, st);
}
