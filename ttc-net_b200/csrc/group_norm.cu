// Group norm over the channels of each row (a token's heads), with an activation or a gate, and
// its backward.  Row r, group G of n channels, c a channel of it:
//   xhat = (x - mean_G) rstd_G,  rstd_G = rsqrt(var_G + eps)      (fp32, variance about the mean)
//   z = xhat w_c + b_c
//   y = act(z)  without a gate,   y = z act(gate)  with one
// Backward, from g = dL/dy, with the statistics recomputed from x instead of saved:
//   gz = g act'(z)   or   gz = g act(gate),  dgate = g z act'(gate)
//   dw_c = sum_r gz xhat,  db_c = sum_r gz,  gx = gz w
//   dx = rstd (gx - mean_G(gx) - xhat mean_G(gx xhat))
//
// Bound by memory: every tensor is read or written once.  A group is a segment of SEG lanes of
// a warp holding K vectors of V channels each (16-byte accesses where the addresses allow, else
// V = 1), so its sums are xor shuffles in a fixed order.  A warp keeps its columns and walks down
// the rows: weight and bias are loaded once, and dw, db are accumulated in registers, then over
// the CTA's warps in shared memory, then over the row slabs by group_norm_sum_kernel -- three fixed
// orders, so results repeat bit by bit.
// 16 384 rows of 32 groups of 128 with a silu gate in bf16: forward 84 us (403 MB, 4.8 TB/s), backward 134 us (671 MB,
// 5.0 TB/s) and 4 us for the sum over row slabs.  The statistics' shuffles and the gate's exponentials issue about as long
// as the bytes take, which is what keeps both at 0.75 of the copy rate.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cstdio>
#include <type_traits>

#include "lqr_common.cuh"
#include "ttc_b200.h"

namespace ttc {
int set_error(int code, const char* msg);
}

namespace {

using ttc::ldf;
using ttc::stf;

constexpr int kWarps = 8;

struct GN {
  const void *x, *gate, *w, *b, *g;
  int64_t xs, gs;  // row strides of x and gate
  void *y, *dx, *dgate;
  float* partial;  // [slabs][2][C], null without dw and db
  int64_t rows;
  int groups, n, seg, act, w_f32;
  float eps;
};

// One or two neighbouring channels in fp32; two at a time with the packed instructions (the kernels
// are bound by instructions, not by memory, where each channel takes its own).
template <int V>
struct ElemOf {
  using type = float2;
};
template <>
struct ElemOf<1> {
  using type = float;
};
__device__ __forceinline__ float add(float a, float b) { return a + b; }
__device__ __forceinline__ float mul(float a, float b) { return a * b; }
__device__ __forceinline__ float fma_(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ uint64_t pair(float2 a) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a.x), "f"(a.y));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t r) {
  float2 a;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a.x), "=f"(a.y) : "l"(r));
  return a;
}
__device__ __forceinline__ float2 add(float2 a, float2 b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair(a)), "l"(pair(b)));
  return unpair(r);
}
__device__ __forceinline__ float2 mul(float2 a, float2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair(a)), "l"(pair(b)));
  return unpair(r);
}
__device__ __forceinline__ float2 fma_(float2 a, float2 b, float2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(pair(a)), "l"(pair(b)), "l"(pair(c)));
  return unpair(r);
}
template <typename E>
__device__ __forceinline__ E all(float a) {
  if constexpr (sizeof(E) == 4) {
    return a;
  } else {
    return make_float2(a, a);
  }
}
__device__ __forceinline__ float both(float a) { return a; }
__device__ __forceinline__ float both(float2 a) { return a.x + a.y; }

// V channels as they lie in memory (one, or 16 bytes), and as numbers.
template <int V, typename T>
struct Raw {
  T v;
  __device__ __forceinline__ void load(const T* p, bool on) { v = on ? *p : T(0.f); }
  __device__ __forceinline__ void get(float (&o)[1]) const { o[0] = ldf(&v); }
};
template <typename T>
struct Raw<4, T> {
  float4 v;
  __device__ __forceinline__ void load(const T* p, bool on) {
    v = on ? *reinterpret_cast<const float4*>(p) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  __device__ __forceinline__ void get(float2 (&o)[2]) const { o[0] = make_float2(v.x, v.y), o[1] = make_float2(v.z, v.w); }
};
template <typename T>
struct Raw<8, T> {
  uint4 v;
  __device__ __forceinline__ void load(const T* p, bool on) {
    v = on ? *reinterpret_cast<const uint4*>(p) : make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ void get(float2 (&o)[4]) const {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = make_float2(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u));
  }
};

template <typename T>
__device__ __forceinline__ void put(T* p, const float (&v)[1]) {
  stf(p, v[0]);
}
__device__ __forceinline__ void put(float* p, const float2 (&v)[2]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
}
__device__ __forceinline__ void put(__nv_bfloat16* p, const float2 (&v)[4]) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v[i].x, v[i].y);
    u[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
}

// sigmoid(u).  For bf16 outputs with the approximate exponential and reciprocal, off by up to (4 + 1.2 |u|) 2^-23 (10^-5
// at u = -88, where u sigmoid(u) is 10^-36; the result is rounded to 2^-8); their exact forms were half of the
// kernels' instructions.
template <typename T>
__device__ __forceinline__ float sigmoid(float u) {
  if constexpr (sizeof(T) == 2) {
    return __fdividef(1.f, 1.f + __expf(-u));
  } else {
    return 1.f / (1.f + expf(-u));
  }
}
template <typename T>
__device__ __forceinline__ float2 sigmoid2(float2 u) {
  return make_float2(sigmoid<T>(u.x), sigmoid<T>(u.y));
}
template <typename T>
__device__ __forceinline__ float sigmoid2(float u) {
  return sigmoid<T>(u);
}
// Phi(u) and the normal density.
__device__ __forceinline__ float cdf(float u) { return 0.5f * (1.f + erff(u * 0.70710678118654752f)); }
__device__ __forceinline__ float2 cdf(float2 u) { return make_float2(cdf(u.x), cdf(u.y)); }
__device__ __forceinline__ float pdf(float u) { return 0.3989422804014327f * expf(-0.5f * u * u); }
__device__ __forceinline__ float2 pdf(float2 u) { return make_float2(pdf(u.x), pdf(u.y)); }

// f = act(u) and d = act'(u).
template <int ACT, typename T, typename E>
__device__ __forceinline__ void act_grad(E u, E& f, E& d) {
  if constexpr (ACT == TTC_ACT_SILU) {
    const E p = sigmoid2<T>(u);
    f = mul(u, p);
    // p (1 + u (1 - p)) = p + f (1 - p)
    d = fma_(f, fma_(p, all<E>(-1.f), all<E>(1.f)), p);
  } else if constexpr (ACT == TTC_ACT_GELU) {
    const E c = cdf(u);
    f = mul(u, c);
    d = fma_(u, pdf(u), c);
  } else {
    f = u;
    d = all<E>(1.f);
  }
}
template <int ACT, typename T, typename E>
__device__ __forceinline__ E act_of(E u) {
  if constexpr (ACT == TTC_ACT_SILU) return mul(u, sigmoid2<T>(u));
  if constexpr (ACT == TTC_ACT_GELU) return mul(u, cdf(u));
  return u;
}
// f(activation, whether there is a gate), both as compile-time constants: one branch for a whole row.
template <typename F>
__device__ __forceinline__ void with_kind(int act, bool gated, F&& f) {
  using std::integral_constant;
  if (act == TTC_ACT_SILU) {
    if (gated)
      f(integral_constant<int, TTC_ACT_SILU>{}, std::true_type{});
    else
      f(integral_constant<int, TTC_ACT_SILU>{}, std::false_type{});
  } else if (act == TTC_ACT_GELU) {
    if (gated)
      f(integral_constant<int, TTC_ACT_GELU>{}, std::true_type{});
    else
      f(integral_constant<int, TTC_ACT_GELU>{}, std::false_type{});
  } else {
    if (gated)
      f(integral_constant<int, TTC_ACT_NONE>{}, std::true_type{});
    else
      f(integral_constant<int, TTC_ACT_NONE>{}, std::false_type{});
  }
}

// Sum over the SEG lanes of a group (SEG = 0: `seg` of them).
template <int SEG>
__device__ __forceinline__ float seg_sum(float v, int seg) {
  if constexpr (SEG > 0) {
#pragma unroll
    for (int o = SEG / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  } else {
    for (int o = seg >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  }
  return v;
}

__device__ __forceinline__ float param(const void* p, int f32, bool bf16, int64_t i, float none) {
  if (p == nullptr) return none;
  return !bf16 || f32 ? static_cast<const float*>(p)[i] : ldf(static_cast<const __nv_bfloat16*>(p) + i);
}

// Deviations from the mean (0 beyond the group) and rstd of the group held in x.
template <int SEG, int K, typename E, int N>
__device__ __forceinline__ float normalise(E (&x)[K][N], const bool (&on)[K], int seg, float inv_n, float eps) {
  E s = all<E>(0.f);
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < N; ++i) s = add(s, x[k][i]);
  const E mean = all<E>(-seg_sum<SEG>(both(s), seg) * inv_n);
  E q = all<E>(0.f);
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      x[k][i] = on[k] ? add(x[k][i], mean) : all<E>(0.f);
      q = fma_(x[k][i], x[k][i], q);
    }
  return rsqrtf(seg_sum<SEG>(both(q), seg) * inv_n + eps);
}

// Weight and bias of a CTA's columns, and where a lane finds its own: element i of vector k at [k N + i][lane].
template <int K, typename E, int N>
struct Params {
  E w[K * N][32], b[K * N][32];
  template <typename T>
  __device__ __forceinline__ void load(const GN& P, const bool (&on)[K], const int64_t (&col)[K]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int PER = sizeof(E) / 4;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (warp == (k * N + i) % kWarps) {
          float v[2][PER];
#pragma unroll
          for (int e = 0; e < PER; ++e) {
            v[0][e] = on[k] ? param(P.w, P.w_f32, sizeof(T) == 2, col[k] + i * PER + e, 1.f) : 0.f;
            v[1][e] = on[k] ? param(P.b, P.w_f32, sizeof(T) == 2, col[k] + i * PER + e, 0.f) : 0.f;
          }
          w[k * N + i][lane] = *reinterpret_cast<const E*>(v[0]);
          b[k * N + i][lane] = *reinterpret_cast<const E*>(v[1]);
        }
    __syncthreads();
  }
};

template <typename T, int V, int K, int SEG>
__global__ void __launch_bounds__(32 * kWarps) group_norm_fwd_kernel(const GN P) {
  using E = typename ElemOf<V>::type;
  constexpr int N = V == 1 ? 1 : V / 2;
  __shared__ __align__(16) Params<K, E, N> par;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int seg = SEG > 0 ? SEG : P.seg;
  const int ls = lane % seg, group = blockIdx.y * (32 / seg) + lane / seg;
  const int64_t C = static_cast<int64_t>(P.groups) * P.n;
  const float inv_n = 1.f / P.n;
  bool on[K];
  int64_t col[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (ls + k * seg) * V;
    on[k] = group < P.groups && c < P.n;
    col[k] = on[k] ? static_cast<int64_t>(group) * P.n + c : 0;
  }
  par.template load<T>(P, on, col);
  const T* gate = static_cast<const T*>(P.gate);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kWarps;
  Raw<V, T> rx[K], rg[K];
  auto fetch = [&](int64_t r) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      rx[k].load(static_cast<const T*>(P.x) + r * P.xs + col[k], on[k]);
      if (gate != nullptr) rg[k].load(gate + r * P.gs + col[k], on[k]);
    }
  };
  constexpr bool AHEAD = K == 1;  // registers for a second row
  int64_t r = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
  if (AHEAD && r < P.rows) fetch(r);
  for (; r < P.rows; r += step) {
    if (!AHEAD) fetch(r);
    E x[K][N], ga[K][N];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      rx[k].get(x[k]);
      if (gate != nullptr) rg[k].get(ga[k]);
    }
    if (AHEAD && r + step < P.rows) fetch(r + step);  // the next row's loads under this one's arithmetic
    const E rstd = all<E>(normalise<SEG>(x, on, seg, inv_n, P.eps));
    with_kind(P.act, gate != nullptr, [&](auto act, auto gated) {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const E z = fma_(mul(x[k][i], rstd), par.w[k * N + i][lane], par.b[k * N + i][lane]);
          if constexpr (decltype(gated)::value)
            x[k][i] = mul(z, act_of<decltype(act)::value, T>(ga[k][i]));
          else
            x[k][i] = act_of<decltype(act)::value, T>(z);
        }
    });
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (on[k]) put(static_cast<T*>(P.y) + r * C + col[k], x[k]);
  }
}

template <typename T, int V, int K, int SEG>
__global__ void __launch_bounds__(32 * kWarps, K == 1 ? 2 : 1) group_norm_bwd_kernel(const GN P) {
  using E = typename ElemOf<V>::type;
  constexpr int N = V == 1 ? 1 : V / 2;
  __shared__ __align__(16) Params<K, E, N> par;
  __shared__ __align__(16) E red[kWarps][K * N][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int seg = SEG > 0 ? SEG : P.seg;
  const int ls = lane % seg, group = blockIdx.y * (32 / seg) + lane / seg;
  const int64_t C = static_cast<int64_t>(P.groups) * P.n;
  const float inv_n = 1.f / P.n;
  bool on[K];
  int64_t col[K];
  E dw[K][N], db[K][N];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (ls + k * seg) * V;
    on[k] = group < P.groups && c < P.n;
    col[k] = on[k] ? static_cast<int64_t>(group) * P.n + c : 0;
#pragma unroll
    for (int i = 0; i < N; ++i) dw[k][i] = db[k][i] = all<E>(0.f);
  }
  par.template load<T>(P, on, col);
  const T* gate = static_cast<const T*>(P.gate);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kWarps;
  Raw<V, T> rx[K], rg[K], rd[K];
  auto fetch = [&](int64_t r) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      rx[k].load(static_cast<const T*>(P.x) + r * P.xs + col[k], on[k]);
      rd[k].load(static_cast<const T*>(P.g) + r * C + col[k], on[k]);
      if (gate != nullptr) rg[k].load(gate + r * P.gs + col[k], on[k]);
    }
  };
  int64_t r = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
  constexpr bool AHEAD = K == 1;  // registers for a second row
  if (AHEAD && r < P.rows) fetch(r);
  for (; r < P.rows; r += step) {
    if (!AHEAD) fetch(r);
    E x[K][N], ga[K][N], g[K][N];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      rx[k].get(x[k]);
      rd[k].get(g[k]);
      if (gate != nullptr) rg[k].get(ga[k]);
    }
    if (AHEAD && r + step < P.rows) fetch(r + step);  // the next row's loads under this one's arithmetic
    const float rs = normalise<SEG>(x, on, seg, inv_n, P.eps);
    const E rstd = all<E>(rs);
    // beyond the group g is 0, and so is every sum's part
    E s1 = all<E>(0.f), s2 = all<E>(0.f);
    with_kind(P.act, gate != nullptr, [&](auto act, auto gated) {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const E w = par.w[k * N + i][lane];
          x[k][i] = mul(x[k][i], rstd);
          const E z = fma_(x[k][i], w, par.b[k * N + i][lane]);
          E f, d;
          if constexpr (decltype(gated)::value) {
            act_grad<decltype(act)::value, T>(ga[k][i], f, d);
            ga[k][i] = mul(mul(g[k][i], z), d);
            g[k][i] = mul(g[k][i], f);
          } else {
            act_grad<decltype(act)::value, T>(z, f, d);
            g[k][i] = mul(g[k][i], d);
          }
          dw[k][i] = fma_(g[k][i], x[k][i], dw[k][i]);
          db[k][i] = add(db[k][i], g[k][i]);
          g[k][i] = mul(g[k][i], w);
          s1 = add(s1, g[k][i]);
          s2 = fma_(g[k][i], x[k][i], s2);
        }
    });
    const E m1 = all<E>(-seg_sum<SEG>(both(s1), seg) * inv_n), m2 = all<E>(-seg_sum<SEG>(both(s2), seg) * inv_n);
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int i = 0; i < N; ++i) x[k][i] = mul(rstd, fma_(x[k][i], m2, add(g[k][i], m1)));
      if (on[k]) {
        if (P.dx != nullptr) put(static_cast<T*>(P.dx) + r * C + col[k], x[k]);
        if (P.dgate != nullptr) put(static_cast<T*>(P.dgate) + r * C + col[k], ga[k]);
      }
    }
  }
  if (P.partial == nullptr) return;
  constexpr int PER = sizeof(E) / 4;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < N; ++i) red[warp][k * N + i][lane] = which ? db[k][i] : dw[k][i];
    __syncthreads();
    for (int e = warp; e < K * N; e += kWarps) {
      E s = all<E>(0.f);
#pragma unroll
      for (int u = 0; u < kWarps; ++u) s = add(s, red[u][e][lane]);
      const int c = (ls + (e / N) * seg) * V;  // this lane's vector number e / N
      if (group < P.groups && c < P.n) {
        float* o = P.partial + (static_cast<int64_t>(blockIdx.x) * 2 + which) * C + static_cast<int64_t>(group) * P.n + c +
                   (e % N) * PER;
        const float* v = reinterpret_cast<const float*>(&s);
#pragma unroll
        for (int j = 0; j < PER; ++j) o[j] = v[j];
      }
    }
  }
}

// dw, db: the sums over the slabs of `partial`, 32 columns a CTA, each warp a share of the slabs.
template <typename TW>
__global__ void __launch_bounds__(32 * kWarps) group_norm_sum_kernel(const float* __restrict__ partial, int slabs, int64_t C,
                                                                     TW* dw, TW* db) {
  __shared__ float red[kWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, which = blockIdx.y;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  float s = 0.f;
  if (c < C) {
#pragma unroll 4
    for (int i = warp; i < slabs; i += kWarps) s += partial[(static_cast<int64_t>(i) * 2 + which) * C + c];
  }
  red[warp][lane] = s;
  __syncthreads();
  TW* out = which ? db : dw;
  if (warp != 0 || c >= C || out == nullptr) return;
  s = 0.f;
#pragma unroll
  for (int u = 0; u < kWarps; ++u) s += red[u][lane];
  stf(out + c, s);
}

int fail(int code, const char* msg) { return ttc::set_error(code, msg); }

int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return TTC_OK;
  char buf[256];
  snprintf(buf, sizeof(buf), "%s: %s", what, cudaGetErrorString(e));
  return fail(TTC_ERR_CUDA, buf);
}

int check(int64_t rows, int groups, int n, int act, int dtype) {
  if (rows < 0 || groups < 1 || n < 1) return fail(TTC_ERR_INVALID, "group_norm: sizes must be positive");
  if (groups > 65535) return fail(TTC_ERR_UNSUPPORTED, "group_norm: more than 65535 groups");
  if (n > 1024) return fail(TTC_ERR_UNSUPPORTED, "group_norm: groups of more than 1024 channels");
  if (act < TTC_ACT_NONE || act > TTC_ACT_GELU) return fail(TTC_ERR_INVALID, "group_norm: unknown activation");
  if (dtype != TTC_DTYPE_F32 && dtype != TTC_DTYPE_BF16)
    return fail(TTC_ERR_INVALID, "group_norm: dtype must be TTC_DTYPE_F32 or TTC_DTYPE_BF16");
  return TTC_OK;
}

// Lanes of a group for vectors of v channels.
int seg_of(int n, int v) {
  int seg = 1;
  while (seg < 32 && seg * v < n) seg *= 2;
  return seg;
}

// CTAs along the rows: as many as are resident at once, 2 an SM for the backward, whose slabs of dw and db are
// written and read again (0.6 MB beside 671 MB at 16 384 x 4096 bf16; with 3 an SM, at 80 registers, it took 161 us against 134), 6 an SM for the forward.
int slabs_of(int64_t rows, int groups, int n, int v, int per_sm) {
  const int gpw = 32 / seg_of(n, v);
  const int64_t tiles = (groups + gpw - 1) / gpw;
  // not one CTA more than fit at once: a last wave of a few would cost as much as a full one
  const int64_t want = std::max<int64_t>(1, 148LL * per_sm / tiles);
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(want, (rows + kWarps - 1) / kWarps)));
}
constexpr int kFwdPerSM = 6, kBwdPerSM = 2;

bool vec_ok(const void* p, int64_t stride, int v) {
  return p == nullptr || ((reinterpret_cast<uintptr_t>(p) & 15u) == 0 && stride % v == 0);
}

template <typename T>
int run(GN P, bool backward, void* dw, void* db, cudaStream_t st) {
  constexpr int VT = 16 / sizeof(T);
  const int64_t C = static_cast<int64_t>(P.groups) * P.n;
  const bool vec = P.n % VT == 0 && vec_ok(P.x, P.xs, VT) && vec_ok(P.gate, P.gs, VT) && vec_ok(P.g, C, VT) &&
                   vec_ok(P.y, C, VT) && vec_ok(P.dx, C, VT) && vec_ok(P.dgate, C, VT);
  const int v = vec ? VT : 1;
  P.seg = seg_of(P.n, v);
  const int gpw = 32 / P.seg, per_lane = (P.n + P.seg * v - 1) / (P.seg * v);
  const int slabs = slabs_of(P.rows, P.groups, P.n, v, backward ? kBwdPerSM : kFwdPerSM);
  const dim3 grid(slabs, (P.groups + gpw - 1) / gpw);
#define TTC_GN(V, K, SEG)                                                  \
  do {                                                                     \
    if (backward)                                                          \
      group_norm_bwd_kernel<T, V, K, SEG><<<grid, 32 * kWarps, 0, st>>>(P); \
    else                                                                   \
      group_norm_fwd_kernel<T, V, K, SEG><<<grid, 32 * kWarps, 0, st>>>(P); \
  } while (0)
  if (vec) {
    if (per_lane == 1) {
      switch (P.seg) {
        case 4: TTC_GN(VT, 1, 4); break;
        case 8: TTC_GN(VT, 1, 8); break;
        case 16: TTC_GN(VT, 1, 16); break;
        case 32: TTC_GN(VT, 1, 32); break;
        default: TTC_GN(VT, 1, 0);
      }
    } else if (per_lane <= 4) {
      TTC_GN(VT, 4, 32);
    } else if constexpr (VT == 4) {
      TTC_GN(VT, 8, 32);
    }
  } else if (per_lane <= 4) {
    TTC_GN(1, 4, 0);
  } else {
    TTC_GN(1, 32, 32);
  }
#undef TTC_GN
  if (int rc = launched(backward ? "group_norm_bwd_kernel launch" : "group_norm_fwd_kernel launch")) return rc;
  if (P.partial == nullptr) return TTC_OK;
  const dim3 sgrid(static_cast<unsigned>((C + 31) / 32), 2);
  if (sizeof(T) == 4 || P.w_f32)
    group_norm_sum_kernel<float><<<sgrid, 32 * kWarps, 0, st>>>(P.partial, slabs, C, static_cast<float*>(dw),
                                                                static_cast<float*>(db));
  else
    group_norm_sum_kernel<__nv_bfloat16><<<sgrid, 32 * kWarps, 0, st>>>(
        P.partial, slabs, C, static_cast<__nv_bfloat16*>(dw), static_cast<__nv_bfloat16*>(db));
  return launched("group_norm_sum_kernel launch");
}

}  // namespace

extern "C" int64_t ttc_group_norm_workspace(int64_t rows, int groups, int n, int dtype) {
  if (int rc = check(rows, groups, n, TTC_ACT_NONE, dtype)) return -rc;
  const int v = dtype == TTC_DTYPE_F32 ? 4 : 8;
  // whichever vector width the addresses allow
  const int slabs = std::max(slabs_of(rows, groups, n, v, kBwdPerSM), slabs_of(rows, groups, n, 1, kBwdPerSM));
  return static_cast<int64_t>(slabs) * 2 * groups * n * 4;
}

extern "C" int ttc_group_norm_fwd(const void* x, int64_t x_stride, const void* gate, int64_t gate_stride,
                                  const void* weight, const void* bias, int param_f32, int64_t rows, int groups, int n,
                                  int act, float eps, int dtype, void* y, void* stream) {
  if (int rc = check(rows, groups, n, act, dtype)) return rc;
  if (rows == 0) return TTC_OK;
  if (!x || !y) return fail(TTC_ERR_INVALID, "group_norm_fwd: null pointer");
  GN P{};
  P.x = x, P.xs = x_stride, P.gate = gate, P.gs = gate_stride, P.w = weight, P.b = bias, P.w_f32 = param_f32;
  P.rows = rows, P.groups = groups, P.n = n, P.act = act, P.eps = eps, P.y = y;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == TTC_DTYPE_F32 ? run<float>(P, false, nullptr, nullptr, st)
                                : run<__nv_bfloat16>(P, false, nullptr, nullptr, st);
}

extern "C" int ttc_group_norm_bwd(const void* x, int64_t x_stride, const void* gate, int64_t gate_stride,
                                  const void* weight, const void* bias, int param_f32, const void* g, int64_t rows,
                                  int groups, int n, int act, float eps, int dtype, void* dx, void* dgate, void* dweight,
                                  void* dbias, void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = check(rows, groups, n, act, dtype)) return rc;
  const bool params = dweight != nullptr || dbias != nullptr;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (rows == 0) {  // empty sums
    const size_t bytes = static_cast<size_t>(groups) * n * (dtype == TTC_DTYPE_F32 || param_f32 ? 4 : 2);
    if ((dweight && cudaMemsetAsync(dweight, 0, bytes, st) != cudaSuccess) ||
        (dbias && cudaMemsetAsync(dbias, 0, bytes, st) != cudaSuccess))
      return launched("group_norm_bwd memset");
    return TTC_OK;
  }
  if (!x || !g || (dgate && !gate)) return fail(TTC_ERR_INVALID, "group_norm_bwd: null pointer");
  if (params && (!workspace || workspace_bytes < ttc_group_norm_workspace(rows, groups, n, dtype)))
    return fail(TTC_ERR_INVALID, "group_norm_bwd: workspace missing or smaller than ttc_group_norm_workspace");
  GN P{};
  P.x = x, P.xs = x_stride, P.gate = gate, P.gs = gate_stride, P.w = weight, P.b = bias, P.w_f32 = param_f32, P.g = g;
  P.rows = rows, P.groups = groups, P.n = n, P.act = act, P.eps = eps, P.dx = dx, P.dgate = dgate;
  P.partial = params ? static_cast<float*>(workspace) : nullptr;
  return dtype == TTC_DTYPE_F32 ? run<float>(P, true, dweight, dbias, st) : run<__nv_bfloat16>(P, true, dweight, dbias, st);
}
