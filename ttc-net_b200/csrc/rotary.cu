// Rotary positions: pair p of a head's first 2 half values turns by angle = position * inv_freq[p],
//   (a, b) -> m (a cos - b sin, a sin + b cos),
// pairs (p, p + half) or, interleaved, (2p, 2p + 1); values behind 2 half are copied.  The backward
// is the turn by -angle with the same factor m.
//
// The angle is formed and reduced to [-pi, pi] in 64 bits: at position 10^6 one 32-bit rounding of
// it is 0.03 rad.  A CTA takes a few tokens, computes the cosines and sines of their pairs once
// into shared memory (256 / half tokens, so that a thread has about one pair) and streams the
// heads of q and k past them; bound by memory, each value is read and written once.
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

template <typename T, int V>
__device__ __forceinline__ void load(float (&v)[V], const T* p) {
  if constexpr (V == 1) {
    v[0] = ldf(p);
  } else if constexpr (sizeof(T) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
  } else {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(u[i] << 16);
      v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  }
}
template <typename T, int V>
__device__ __forceinline__ void store(T* p, const float (&v)[V]) {
  if constexpr (V == 1) {
    stf(p, v[0]);
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      u[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
  }
}

// Units of a head: `half / V` (pairs of vectors) or, interleaved, `2 half / V` (vectors of V / 2
// pairs; V = 1 takes a pair as two scalars), then the vectors that are copied.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const Rot P) {
  extern __shared__ float2 cs[];  // [tokens][half]
  __shared__ int64_t offset[kMaxTokens][2];  // of the tokens in q and k
  const int64_t tok0 = static_cast<int64_t>(blockIdx.x) * P.tokens;
  const int64_t total = P.B * P.T;
  const int ntok = static_cast<int>(min(static_cast<int64_t>(P.tokens), total - tok0));
  for (int i = threadIdx.x; i < ntok * P.half; i += kThreads) {
    const int t = i / P.half, p = i - t * P.half;
    const int64_t tok = tok0 + t, b = tok / P.T, off = b * P.pb + (tok - b * P.T) * P.pt;
    const double pos = P.pos64 ? static_cast<double>(static_cast<const int64_t*>(P.pos)[off])
                               : static_cast<double>(static_cast<const int*>(P.pos)[off]);
    const double angle = P.sign * pos * P.inv_freq[p];
    const double turns = rint(angle * 0.15915494309189535);  // 1 / (2 pi)
    // 2 pi as a sum of two doubles, so that the reduction keeps its digits for many turns
    const double r = fma(-turns, 2.4492935982947064e-16, fma(-turns, 6.283185307179586, angle));
    const float rh = static_cast<float>(r), rl = static_cast<float>(r - static_cast<double>(rh));
    float s, c;
    sincosf(rh, &s, &c);
    cs[i] = make_float2(P.mag * fmaf(-s, rl, c), P.mag * fmaf(c, rl, s));
  }
  if (threadIdx.x < 2 * ntok) {
    const int t = threadIdx.x >> 1, w = threadIdx.x & 1;
    const int64_t tok = tok0 + t, b = tok / P.T;
    offset[t][w] = b * P.sb[w] + (tok - b * P.T) * P.st[w];
  }
  __syncthreads();
  const bool pairs_split = V == 1 || !P.interleaved;  // a and b of a pair in different units' vectors
  const int turn = pairs_split ? P.half / V : 2 * P.half / V;
  const int units = turn + (P.D - 2 * P.half) / V;
  const int h0 = blockIdx.y * P.heads, nh = min(P.heads, P.H[0] + P.H[1] - h0);
  // thread -> unit and (token, head); the remaining threads of the last round idle
  const int lanes = min(units, kThreads), step = kThreads / lanes;
  const int lane = threadIdx.x % lanes, r0 = threadIdx.x / lanes;
  if (r0 >= step) return;
  for (int u = lane; u < units; u += lanes) {
    int t = r0 / nh, h = r0 - t * nh;
#pragma unroll 4
    for (int r = r0; r < ntok * nh; r += step) {
      const int hh = h0 + h, which = hh >= P.H[0], head = which ? hh - P.H[0] : hh;
      const T* src = static_cast<const T*>(P.x[which]) + offset[t][which] + head * P.sh[which];
      T* dst = static_cast<T*>(P.y[which]) + ((tok0 + t) * P.H[which] + head) * P.D;
      if (u >= turn) {
        const int c = 2 * P.half + (u - turn) * V;
        float v[V];
        load<T, V>(v, src + c);
        store<T, V>(dst + c, v);
      } else if (pairs_split) {
        const int ia = P.interleaved ? 2 * u : u * V, ib = P.interleaved ? 2 * u + 1 : u * V + P.half;
        float a[V], bb[V];
        load<T, V>(a, src + ia);
        load<T, V>(bb, src + ib);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float2 w = cs[t * P.half + u * V + i];
          const float x = a[i], y = bb[i];
          a[i] = fmaf(x, w.x, -y * w.y);
          bb[i] = fmaf(x, w.y, y * w.x);
        }
        store<T, V>(dst + ia, a);
        store<T, V>(dst + ib, bb);
      } else if constexpr (V > 1) {
        float a[V];
        load<T, V>(a, src + u * V);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
          const float2 w = cs[t * P.half + u * (V / 2) + i];
          const float x = a[2 * i], y = a[2 * i + 1];
          a[2 * i] = fmaf(x, w.x, -y * w.y);
          a[2 * i + 1] = fmaf(x, w.y, y * w.x);
        }
        store<T, V>(dst + u * V, a);
      }
      h += step;
      while (h >= nh) {
        h -= nh;
        ++t;
      }
    }
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
  if (vec)
    rotary_kernel<T, VT><<<grid, kThreads, smem, st>>>(P);
  else
    rotary_kernel<T, 1><<<grid, kThreads, smem, st>>>(P);
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
