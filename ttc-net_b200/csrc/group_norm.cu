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

// V channels as they lie in memory (one, or 16 bytes), and as floats.
template <int V, typename T>
struct Raw {
  T v;
  __device__ __forceinline__ void load(const T* p, bool on) { v = on ? *p : T(0.f); }
  __device__ __forceinline__ void floats(float (&o)[V]) const { o[0] = ldf(&v); }
};
template <typename T>
struct Raw<4, T> {
  float4 v;
  __device__ __forceinline__ void load(const T* p, bool on) {
    v = on ? *reinterpret_cast<const float4*>(p) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  __device__ __forceinline__ void floats(float (&o)[4]) const { o[0] = v.x, o[1] = v.y, o[2] = v.z, o[3] = v.w; }
};
template <typename T>
struct Raw<8, T> {
  uint4 v;
  __device__ __forceinline__ void load(const T* p, bool on) {
    v = on ? *reinterpret_cast<const uint4*>(p) : make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ void floats(float (&o)[8]) const {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o[2 * i] = __uint_as_float(u[i] << 16);
      o[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  }
};

template <int V, typename T>
__device__ __forceinline__ void st_vec(T* p, const float (&v)[V]) {
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

// sigmoid(u).  For bf16 outputs with the approximate exponential and reciprocal, off by a few 2^-22 (the
// result is rounded to 2^-8); their exact forms are half of the kernels' instructions.
template <typename T>
__device__ __forceinline__ float sigmoid(float u) {
  if constexpr (sizeof(T) == 2) {
    return __fdividef(1.f, 1.f + __expf(-u));
  } else {
    return 1.f / (1.f + expf(-u));
  }
}
// act(u) and act'(u).
template <typename T>
__device__ __forceinline__ void act_grad(int act, float u, float& f, float& d) {
  if (act == TTC_ACT_SILU) {
    const float p = sigmoid<T>(u);
    f = u * p;
    d = p * (1.f + u * (1.f - p));
  } else if (act == TTC_ACT_GELU) {
    const float c = 0.5f * (1.f + erff(u * 0.70710678118654752f));
    f = u * c;
    d = c + u * 0.3989422804014327f * expf(-0.5f * u * u);
  } else {
    f = u;
    d = 1.f;
  }
}
template <typename T>
__device__ __forceinline__ float act_of(int act, float u) {
  if (act == TTC_ACT_SILU) return u * sigmoid<T>(u);
  if (act == TTC_ACT_GELU) return 0.5f * u * (1.f + erff(u * 0.70710678118654752f));
  return u;
}

__device__ __forceinline__ float seg_sum(float v, int seg) {
  for (int o = seg >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ float param(const void* p, int f32, bool bf16, int64_t i, float none) {
  if (p == nullptr) return none;
  return !bf16 || f32 ? static_cast<const float*>(p)[i] : ldf(static_cast<const __nv_bfloat16*>(p) + i);
}

// Deviations from the mean (0 beyond the group) and rstd of the group held in x.
template <int V, int K>
__device__ __forceinline__ float normalise(float (&x)[K][V], const bool (&on)[K], int seg, float inv_n, float eps) {
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) s += x[k][i];
  const float mean = seg_sum(s, seg) * inv_n;
  float q = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      x[k][i] = on[k] ? x[k][i] - mean : 0.f;
      q = fmaf(x[k][i], x[k][i], q);
    }
  return rsqrtf(seg_sum(q, seg) * inv_n + eps);
}

template <typename T, int V, int K>
__global__ void __launch_bounds__(32 * kWarps) group_norm_fwd_kernel(const GN P) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int ls = lane % P.seg, group = blockIdx.y * (32 / P.seg) + lane / P.seg;
  const int64_t C = static_cast<int64_t>(P.groups) * P.n;
  const float inv_n = 1.f / P.n;
  bool on[K];
  int64_t col[K];
  float w[K][V], b[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (ls + k * P.seg) * V;
    on[k] = group < P.groups && c < P.n;
    col[k] = on[k] ? static_cast<int64_t>(group) * P.n + c : 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      w[k][i] = on[k] ? param(P.w, P.w_f32, sizeof(T) == 2, col[k] + i, 1.f) : 0.f;
      b[k][i] = on[k] ? param(P.b, P.w_f32, sizeof(T) == 2, col[k] + i, 0.f) : 0.f;
    }
  }
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
  int64_t r = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
  constexpr bool AHEAD = K == 1;  // registers for a second row
  if (AHEAD && r < P.rows) fetch(r);
  for (; r < P.rows; r += step) {
    if (!AHEAD) fetch(r);
    float x[K][V], ga[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      rx[k].floats(x[k]);
      if (gate != nullptr) rg[k].floats(ga[k]);
    }
    if (AHEAD && r + step < P.rows) fetch(r + step);  // the next row's loads under this one's arithmetic
    const float rstd = normalise<V, K>(x, on, P.seg, inv_n, P.eps);
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float z = fmaf(x[k][i] * rstd, w[k][i], b[k][i]);
        x[k][i] = gate != nullptr ? z * act_of<T>(P.act, ga[k][i]) : act_of<T>(P.act, z);
      }
      if (on[k]) st_vec<V>(static_cast<T*>(P.y) + r * C + col[k], x[k]);
    }
  }
}

template <typename T, int V, int K>
__global__ void __launch_bounds__(32 * kWarps) group_norm_bwd_kernel(const GN P) {
  __shared__ float red[kWarps][32 * K * V];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int ls = lane % P.seg, group = blockIdx.y * (32 / P.seg) + lane / P.seg;
  const int64_t C = static_cast<int64_t>(P.groups) * P.n;
  const float inv_n = 1.f / P.n;
  bool on[K];
  int64_t col[K];
  float w[K][V], b[K][V], dw[K][V], db[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (ls + k * P.seg) * V;
    on[k] = group < P.groups && c < P.n;
    col[k] = on[k] ? static_cast<int64_t>(group) * P.n + c : 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      w[k][i] = on[k] ? param(P.w, P.w_f32, sizeof(T) == 2, col[k] + i, 1.f) : 0.f;
      b[k][i] = on[k] ? param(P.b, P.w_f32, sizeof(T) == 2, col[k] + i, 0.f) : 0.f;
      dw[k][i] = db[k][i] = 0.f;
    }
  }
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
    float x[K][V], ga[K][V], g[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      rx[k].floats(x[k]);
      rd[k].floats(g[k]);
      if (gate != nullptr) rg[k].floats(ga[k]);
    }
    if (AHEAD && r + step < P.rows) fetch(r + step);  // the next row's loads under this one's arithmetic
    const float rstd = normalise<V, K>(x, on, P.seg, inv_n, P.eps);
    float m1 = 0.f, m2 = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float xh = x[k][i] * rstd, z = fmaf(xh, w[k][i], b[k][i]);
        float f, d;
        if (gate != nullptr) {
          act_grad<T>(P.act, ga[k][i], f, d);
          ga[k][i] = g[k][i] * z * d;
          g[k][i] *= f;
        } else {
          act_grad<T>(P.act, z, f, d);
          g[k][i] *= d;
        }
        x[k][i] = xh;
        if (on[k]) {
          dw[k][i] = fmaf(g[k][i], xh, dw[k][i]);
          db[k][i] += g[k][i];
        }
        g[k][i] = on[k] ? g[k][i] * w[k][i] : 0.f;
        m1 += g[k][i];
        m2 = fmaf(g[k][i], xh, m2);
      }
    m1 = seg_sum(m1, P.seg) * inv_n;
    m2 = seg_sum(m2, P.seg) * inv_n;
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int i = 0; i < V; ++i) x[k][i] = rstd * (g[k][i] - m1 - x[k][i] * m2);
      if (on[k]) {
        if (P.dx != nullptr) st_vec<V>(static_cast<T*>(P.dx) + r * C + col[k], x[k]);
        if (P.dgate != nullptr) st_vec<V>(static_cast<T*>(P.dgate) + r * C + col[k], ga[k]);
      }
    }
  }
  if (P.partial == nullptr) return;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) red[warp][(k * V + i) * 32 + lane] = which ? db[k][i] : dw[k][i];
    __syncthreads();
    for (int e = warp; e < K * V; e += kWarps) {
      float s = 0.f;
#pragma unroll
      for (int u = 0; u < kWarps; ++u) s += red[u][e * 32 + lane];
      const int c = (ls + (e / V) * P.seg) * V;  // this lane's vector number e / V
      if (group < P.groups && c < P.n)
        P.partial[(static_cast<int64_t>(blockIdx.x) * 2 + which) * C + static_cast<int64_t>(group) * P.n + c + e % V] = s;
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

// CTAs along the rows.  About 4 CTAs an SM in all for the backward, whose slabs of dw and db are
// written and read again (1.2 MB of 537 MB at 16 384 x 4096 bf16); 8 an SM for the forward.
int slabs_of(int64_t rows, int groups, int n, int v, int per_sm) {
  const int gpw = 32 / seg_of(n, v);
  const int64_t tiles = (groups + gpw - 1) / gpw;
  const int64_t want = std::max<int64_t>(1, (148LL * per_sm + tiles - 1) / tiles);
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(want, (rows + kWarps - 1) / kWarps)));
}
constexpr int kFwdPerSM = 8, kBwdPerSM = 4;

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
#define TTC_GN(V, K)                                                  \
  do {                                                                \
    if (backward)                                                     \
      group_norm_bwd_kernel<T, V, K><<<grid, 32 * kWarps, 0, st>>>(P); \
    else                                                              \
      group_norm_fwd_kernel<T, V, K><<<grid, 32 * kWarps, 0, st>>>(P); \
  } while (0)
  if (vec) {
    if (per_lane == 1)
      TTC_GN(VT, 1);
    else if (per_lane <= 4)
      TTC_GN(VT, 4);
    else if constexpr (VT == 4)
      TTC_GN(VT, 8);
  } else if (per_lane <= 4) {
    TTC_GN(1, 4);
  } else {
    TTC_GN(1, 32);
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
