// C entry points of the attention with a fixed decay for each head (decay_attn.cuh has the
// mathematics): how the work is split, the joining of the segments' states, the sum of shared
// heads' gradients, and the kernel for single tokens.
#include <algorithm>

#include "decay_attn_launch.cuh"

namespace ttc {
namespace da {
namespace {

int fail(int code, const char* msg) { return set_error(code, msg); }

int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return TTC_OK;
  char buf[256];
  snprintf(buf, sizeof(buf), "%s: %s", what, cudaGetErrorString(e));
  return fail(TTC_ERR_CUDA, buf);
}

// Segments' own sums -> states at the segments' starts, in place, and the last state:
// run' = gamma^len run + sum.  One thread for each element of a (sequence, head)'s state.
__global__ void __launch_bounds__(256) segment_scan_kernel(const __grid_constant__ Args A) {
  const Pass& P = A.pass[blockIdx.z];
  const int n = blockIdx.y / A.H, h = blockIdx.y % A.H;
  const int size = P.kd * P.vd;
  const int e = blockIdx.x * blockDim.x + threadIdx.x;
  // the first item of this sequence: the segments of the ones before it
  __shared__ int64_t s_first, s_len;
  __shared__ float s_pow[2];  // of a whole segment and of the last one: once a CTA, an exponential in 64 bits is slow
  if (threadIdx.x < 32) {
    int64_t first = 0, row0 = 0, len = A.T;
    if (A.cu == nullptr) {
      first = static_cast<int64_t>(n) * A.n_seg;
    } else {
      for (int i = threadIdx.x; i < n; i += 32) {
        seq_range(A, i, row0, len);
        first += segs_of(A, len);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) first += __shfl_xor_sync(0xffffffffu, first, o);
      seq_range(A, n, row0, len);
    }
    if (threadIdx.x == 0) {
      s_first = first;
      s_len = len;
    }
    const int64_t last = len - static_cast<int64_t>(segs_of(A, len) - 1) * A.seg_len;
    if (threadIdx.x < 2) s_pow[threadIdx.x] = decay_pow(A.log_gamma[h], threadIdx.x ? last : A.seg_len);
  }
  __syncthreads();
  if (e >= size) return;
  const int64_t first = s_first, len = s_len;
  const int segs = segs_of(A, len);
  if (first + segs > A.items) return;  // offsets that are not increasing: more segments than were launched
  const int64_t sbase = (static_cast<int64_t>(n) * A.H + h) * size;
  float run = P.init != nullptr ? P.init[sbase + (e / P.vd) * P.isk + (e % P.vd) * P.isv] : 0.f;
  for (int s = 0; s < segs; ++s) {
    float* p = P.seg + ((first + s) * A.H + h) * size + e;
    if (s + 1 < segs) {
      const float u = *p;
      *p = run;
      run = fmaf(s_pow[0], run, u);
    } else {
      const float u = P.fin != nullptr ? *p : 0.f;
      *p = run;
      if (P.fin != nullptr) P.fin[sbase + e] = fmaf(s_pow[1], run, u);
    }
  }
}

// out[r, hk, d] = sum over the `grp` heads that share hk of in[r, hk grp + j, d], in order;
// blockIdx.y picks one of two (in, out) pairs.
template <typename T>
__global__ void __launch_bounds__(256) shared_heads_kernel(const float* __restrict__ in0, T* __restrict__ out0,
                                                           const float* __restrict__ in1, T* __restrict__ out1,
                                                           int64_t rows_heads, int grp, int d) {
  const float* in = blockIdx.y ? in1 : in0;
  T* out = blockIdx.y ? out1 : out0;
  const int64_t n4 = rows_heads * d / 4;
  for (int64_t x = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; x < n4;
       x += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t rh = x * 4 / d;
    const int c = static_cast<int>(x * 4 - rh * d);
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int j = 0; j < grp; ++j) {
      const float4 v = *reinterpret_cast<const float4*>(in + (rh * grp + j) * d + c);
      s.x += v.x;
      s.y += v.y;
      s.z += v.z;
      s.w += v.w;
    }
    T* o = out + rh * d + c;
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(o) = s;
    } else {
      *reinterpret_cast<uint2*>(o) = make_uint2(mma::pack2(s.x, s.y), mma::pack2(s.z, s.w));
    }
  }
}

// One token for each row b over a cache of states: S = gamma S + k^T v in place, o = scale q S.
// Bound by the state's bytes, read and written once: a thread owns four neighbouring columns
// of every R-th state row (16-byte accesses, up to 8 loads in flight), the rows' parts of o are
// added in shared memory.  Rows of one slot are consecutive tokens of it: the CTA of the first
// such row takes them all in order and the others leave, so no two CTAs touch one state.
// 64 rows of 32 heads of 128 x 128 (268 MB of states): 49 us, 5.5 TB/s or 0.84 of the copy rate.
template <typename T>
__global__ void __launch_bounds__(256)
    decay_attn_step_kernel(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v, int64_t qsb,
                           int64_t qsh, int64_t ksb, int64_t ksh, int64_t vsb, int64_t vsh,
                           const float* __restrict__ log_gamma, float scale, float* state, int64_t slot_stride,
                           const int* __restrict__ slots, int B, int n_slots, int H, int grp, int dk, int dv, int tile,
                           T* __restrict__ o) {
  constexpr int U = 8;
  __shared__ float sq[128], sk[128];
  __shared__ float4 part[256];
  const int tid = threadIdx.x;
  const int h = blockIdx.y, c0 = blockIdx.z * tile;
  int b = blockIdx.x;
  const int lanes = tile / 4, R = 256 / lanes;
  const int r0 = tid / lanes, c = c0 + (tid % lanes) * 4;
  const bool on = r0 < R && c < dv;
  const int slot = slots != nullptr ? slots[b] : b;
  if (slot < 0 || slot >= n_slots) {  // a padding row
    if (on && r0 == 0)
      for (int x = 0; x < 4; ++x) stf(o + (static_cast<int64_t>(b) * H + h) * dv + c + x, 0.f);
    return;
  }
  float* const S = state + slot * slot_stride + static_cast<int64_t>(h) * dk * dv + c;
  auto load = [&](float4(&s)[U], int r) {
#pragma unroll
    for (int x = 0; x < U; ++x) {
      const int rr = r + x * R;
      s[x] = on && rr < dk ? *reinterpret_cast<const float4*>(S + static_cast<int64_t>(rr) * dv)
                           : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  };
  float4 s[U];
  load(s, r0);  // in flight during the search below
  bool later = false;
  if (slots != nullptr && B > 1) {
    bool before = false;
    for (int x = tid; x < B; x += 256) {
      const bool same = slots[x] == slot;
      before |= same && x < b;
      later |= same && x > b;
    }
    if (__syncthreads_or(before)) return;
    later = __syncthreads_or(later);
  }
  const float gamma = decay_pow(log_gamma[h], 1);
  bool loaded = true;
  for (;;) {
    if (tid < dk) {
      sq[tid] = ldf(q + b * qsb + (h / grp) * qsh + tid) * scale;
      sk[tid] = ldf(k + b * ksb + (h / grp) * ksh + tid);
    }
    float4 vv = make_float4(0.f, 0.f, 0.f, 0.f);
    if (on) {
      const T* vp = v + b * vsb + h * vsh + c;
      vv = make_float4(ldf(vp), ldf(vp + 1), ldf(vp + 2), ldf(vp + 3));
    }
    __syncthreads();
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int r = r0; r < dk; r += U * R) {
      if (!loaded) load(s, r);
      loaded = false;
#pragma unroll
      for (int x = 0; x < U; ++x) {
        const int rr = r + x * R;
        if (on && rr < dk) {
          const float kk = sk[rr], qq = sq[rr];
          s[x].x = fmaf(gamma, s[x].x, kk * vv.x);
          s[x].y = fmaf(gamma, s[x].y, kk * vv.y);
          s[x].z = fmaf(gamma, s[x].z, kk * vv.z);
          s[x].w = fmaf(gamma, s[x].w, kk * vv.w);
          *reinterpret_cast<float4*>(S + static_cast<int64_t>(rr) * dv) = s[x];
          acc.x = fmaf(qq, s[x].x, acc.x);
          acc.y = fmaf(qq, s[x].y, acc.y);
          acc.z = fmaf(qq, s[x].z, acc.z);
          acc.w = fmaf(qq, s[x].w, acc.w);
        }
      }
    }
    part[tid] = acc;
    __syncthreads();
    if (on && r0 == 0) {
      for (int r = 1; r < R; ++r) {
        const float4 p = part[tid + r * lanes];
        acc.x += p.x;
        acc.y += p.y;
        acc.z += p.z;
        acc.w += p.w;
      }
      T* op = o + (static_cast<int64_t>(b) * H + h) * dv + c;
      stf(op, acc.x);
      stf(op + 1, acc.y);
      stf(op + 2, acc.z);
      stf(op + 3, acc.w);
    }
    if (!later) return;
    do {
      ++b;
    } while (b < B && slots[b] != slot);
    if (b >= B) return;
    loaded = false;
    __syncthreads();
  }
}

struct Plan {
  int seg_len, n_seg, items;
};

// How a call is split: one CTA for each (sequence, head, pass), or sequences cut into segments whose states
// are summed first (a second pass over k and v) and joined by a scan.  The least cost over the number of segments decides,
// segments have at least four blocks.  In units of a block's time on one CTA (1.9 us in bf16 at 128 x 128, 1.5 at
// 64 x 64; in fp32 7 us at 32 x 64, 9 at 64 x 64; one set of costs for all
// widths), `rounds` of CTAs over the SMs cost their segment's blocks and
// `start` for a CTA's beginning and end; those of the sums `sum` of the blocks and `sum_start`; `more` is for the two
// further launches, `state` for the trips of one segment's 128 x 128 state through memory.  Fitted to measured times: 8192
// tokens, 32 heads of 128: 224 us as one, 134 in 4 segments, 187 in 9; 2 x 4096: 116 as one, 129 in 2.  A backward counts as one
// launch of three passes, also where unequal widths of dk and dv make it two, of 2 / 3 and 1 / 3 of the CTAs.  Packed rows are cut
// by their number alone, the lengths being on the device: one long prompt among three short ones, 32 heads of 128,
// 32 768 tokens, is not (957 us).
struct Costs {
  double start, sum, sum_start, more, state;
};
constexpr Costs kCostsBf16 = {3, 0.75, 4, 5, 0.03}, kCostsF32 = {0, 0.4, 0, 2, 0};

Plan plan(int64_t T, int n_seq, bool packed, int H, int dk, int dv, int passes, int dtype) {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
    (void)cudaGetLastError();
    sms = 148;
  }
  const int64_t rows = static_cast<int64_t>(n_seq) * H * passes;
  // fp32 heads of at most 32 x 32 leave room for two CTAs on an SM (16 x 512 tokens, 32 heads: backward 471 -> 395 us;
  // at 32 x 64 the halved registers cost more than the second CTA gives, 239 -> 308)
  const bool two = dtype == TTC_DTYPE_F32 && width_class_f32(dk) + width_class_f32(dv) <= 64;
  const int64_t slots = two ? 2 * sms : sms;
  const int64_t blocks = (T + C - 1) / C;
  int64_t len = T;
  if (packed) {
    // the lengths are on the device: equal shares of all tokens, where there are CTAs to spare for them
    if (2 * rows <= slots) len = std::max<int64_t>(8 * C, (T * H * passes + slots - rows - 1) / (slots - rows));
  } else if (rows > 0 && rows <= slots) {
    const auto rounds = [&](int64_t ctas) { return static_cast<double>((ctas + slots - 1) / slots); };
    const Costs c = dtype == TTC_DTYPE_BF16 ? kCostsBf16 : kCostsF32;
    double best = static_cast<double>(blocks) + c.start;
    for (int64_t n = 2; n <= blocks / 4 && n <= 2 * slots / rows; ++n) {
      const int64_t each = (blocks + n - 1) / n, used = (blocks + each - 1) / each;
      const double cost = rounds(rows * used) * (each + c.start) + rounds(rows * (used - 1)) * (c.sum * each + c.sum_start) +
                          c.more + c.state * static_cast<double>(rows * used) * dk * dv / 16384;
      if (cost < best) {
        best = cost;
        len = each * C;
      }
    }
  }
  Plan p;
  p.seg_len = static_cast<int>(std::max<int64_t>(C, (len + C - 1) / C * C));
  p.n_seg = static_cast<int>(std::max<int64_t>(1, (T + p.seg_len - 1) / p.seg_len));
  p.items = packed ? static_cast<int>(T / p.seg_len + n_seq) : n_seq * p.n_seg;
  return p;
}

// Whether any sequence may have more than one segment.
bool segmented(const Plan& p, int64_t T) { return p.seg_len < T; }

int check(int64_t T, int n_seq, bool packed, int H, int Hk, int dk, int dv, int dtype) {
  if (T < 0 || T > 0x7fffffffLL - C || n_seq < 0)
    return fail(TTC_ERR_INVALID, "decay_attn: tokens must be in [0, 2^31 - 64), sequences >= 0");
  if (H < 1 || H > 65535 || Hk < 1 || H % Hk != 0)
    return fail(TTC_ERR_INVALID, "decay_attn: heads must be in [1, 65535] and a multiple of the key heads");
  if (dtype != TTC_DTYPE_F32 && dtype != TTC_DTYPE_BF16)
    return fail(TTC_ERR_INVALID, "decay_attn: dtype must be TTC_DTYPE_F32 or TTC_DTYPE_BF16");
  if (dk < 8 || dk > 128 || dk % 8 || dv < 8 || dv > 128 || dv % 8)
    return fail(TTC_ERR_UNSUPPORTED, "decay_attn: head dims must be multiples of 8 from 8 to 128");
  if (static_cast<int64_t>(n_seq) * H > 65535 * 16LL)
    return fail(TTC_ERR_INVALID, "decay_attn: too many sequences x heads (at most 2^20 - 16)");
  // (a packed row of 2^31 tokens has 2^25 blocks and at most one more for each sequence)
  if (!packed && (T / C + 1) * n_seq > 0x7fffffffLL)
    return fail(TTC_ERR_INVALID, "decay_attn: too many blocks of 64 tokens (at most 2^31 - 1)");
  return TTC_OK;
}

bool misaligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

int check_operand(const void* p, const int64_t* s, int n, int dtype) {
  if (misaligned16(p)) return fail(TTC_ERR_INVALID, "decay_attn: q, k, v and g_o must be 16-byte aligned");
  const int unit = dtype == TTC_DTYPE_BF16 ? 8 : 4;
  for (int i = 0; i < n; ++i)
    if (s[i] % unit) return fail(TTC_ERR_INVALID, "decay_attn: strides must be multiples of 16 bytes");
  return TTC_OK;
}

int64_t state_bytes(const Plan& p, int64_t T, int H, int dk, int dv, int passes) {
  return segmented(p, T) ? static_cast<int64_t>(p.items) * H * dk * dv * 4 * passes : 0;
}

int run_passes(Args& A, const Pass* pass, int n, int dtype, bool seg, int* status, cudaStream_t st) {
  const auto go = [&](const Args& a, int m, bool state_only) {
    return dtype == TTC_DTYPE_BF16 ? launch_bf16(a, m, state_only, status, st) : launch_f32(a, m, state_only, st);
  };
  const auto width = dtype == TTC_DTYPE_BF16 ? width_class_bf16 : width_class_f32;
  const auto same = [&](const Pass& x, const Pass& y) {
    return width(x.kd) == width(y.kd) && width(x.vd) == width(y.vd);
  };
  for (int phase = seg ? 0 : 2; phase < 3; ++phase) {
    if (phase == 1) {
      for (int i = 0; i < n; ++i) A.pass[i] = pass[i];
      const dim3 grid((pass[0].kd * pass[0].vd + 255) / 256, A.n_seq * A.H, n);
      segment_scan_kernel<<<grid, 256, 0, st>>>(A);
      if (int rc = launched("segment_scan_kernel launch")) return rc;
      continue;
    }
    bool done[3] = {false, false, false};
    for (int i = 0; i < n; ++i) {
      if (done[i]) continue;
      int m = 0;
      for (int j = i; j < n; ++j)
        if (!done[j] && same(pass[i], pass[j])) {
          A.pass[m++] = pass[j];
          done[j] = true;
        }
      if (int rc = go(A, m, phase == 0)) return rc;
    }
  }
  return TTC_OK;
}

}  // namespace
}  // namespace da
}  // namespace ttc

using namespace ttc;

extern "C" int64_t ttc_decay_attn_workspace(int64_t T, int n_seq, int packed, int H, int Hk, int dk, int dv, int dtype,
                                            int backward) {
  if (int rc = da::check(T, n_seq, packed != 0, H, Hk, dk, dv, dtype)) return -rc;
  if (n_seq == 0) return 0;
  const int passes = backward ? 3 : 1;
  int64_t bytes = da::state_bytes(da::plan(T, n_seq, packed != 0, H, dk, dv, passes, dtype), T, H, dk, dv, passes);
  if (backward && H != Hk) bytes += 2 * (packed ? 1 : n_seq) * T * H * dk * 4;
  return bytes;
}

extern "C" int ttc_decay_attn_fwd(const void* q, const void* k, const void* v, const int64_t* strides,
                                  const float* log_gamma, float scale, const float* initial_state,
                                  const int* cu_seqlens, int64_t T, int n_seq, int H, int Hk, int dk, int dv, int dtype,
                                  void* o, float* final_state, void* workspace, int64_t workspace_bytes, int* status,
                                  void* stream) {
  if (int rc = da::check(T, n_seq, cu_seqlens != nullptr, H, Hk, dk, dv, dtype)) return rc;
  if (n_seq == 0) return cu_seqlens ? da::fail(TTC_ERR_INVALID, "decay_attn: packed rows need a sequence") : TTC_OK;
  if (!strides || !log_gamma || (T > 0 && (!q || !k || !v || !o)))
    return da::fail(TTC_ERR_INVALID, "decay_attn_fwd: null pointer");
  const void* ops[3] = {q, k, v};
  for (int i = 0; i < 3; ++i)
    if (int rc = da::check_operand(ops[i], strides + 3 * i, 3, dtype)) return rc;
  if (da::misaligned16(o)) return da::fail(TTC_ERR_INVALID, "decay_attn_fwd: o must be 16-byte aligned");
  const da::Plan p = da::plan(T, n_seq, cu_seqlens != nullptr, H, dk, dv, 1, dtype);
  const int64_t need = da::state_bytes(p, T, H, dk, dv, 1);
  if (workspace_bytes < need || (need > 0 && (!workspace || da::misaligned16(workspace))))
    return da::fail(TTC_ERR_INVALID, "decay_attn_fwd: workspace missing, misaligned or smaller than ttc_decay_attn_workspace");
  if (T == 0 && final_state == nullptr) return TTC_OK;
  da::Args A{};
  A.log_gamma = log_gamma;
  A.cu = cu_seqlens;
  A.T = T;
  A.n_seq = n_seq;
  A.H = H;
  A.seg_len = p.seg_len;
  A.n_seg = p.n_seg;
  A.items = p.items;
  A.parts = final_state ? 3 : 2;
  da::Pass f{};
  f.q = q, f.k = k, f.v = v;
  for (int i = 0; i < 3; ++i) f.qs[i] = strides[i], f.ks[i] = strides[3 + i], f.vs[i] = strides[6 + i];
  f.qg = f.kg = H / Hk, f.vg = 1;
  f.o = o, f.o_f32 = dtype == TTC_DTYPE_F32;
  f.init = initial_state, f.isk = dv, f.isv = 1;
  f.fin = final_state;
  f.seg = da::segmented(p, T) ? static_cast<float*>(workspace) : nullptr;
  f.kd = dk, f.vd = dv;
  f.a = f.b = scale, f.u = 1.f;
  return da::run_passes(A, &f, 1, dtype, f.seg != nullptr, status,
                        static_cast<cudaStream_t>(stream));
}

extern "C" int ttc_decay_attn_bwd(const void* q, const void* k, const void* v, const int64_t* strides, const void* g_o,
                                  const float* log_gamma, float scale, const float* initial_state,
                                  const float* g_final_state, const int* cu_seqlens, int64_t T, int n_seq, int H, int Hk,
                                  int dk, int dv, int dtype, void* d_q, void* d_k, void* d_v, float* d_initial_state,
                                  void* workspace, int64_t workspace_bytes, int* status, void* stream) {
  if (int rc = da::check(T, n_seq, cu_seqlens != nullptr, H, Hk, dk, dv, dtype)) return rc;
  if (n_seq == 0) return cu_seqlens ? da::fail(TTC_ERR_INVALID, "decay_attn: packed rows need a sequence") : TTC_OK;
  if (!strides || !log_gamma || (T > 0 && (!q || !k || !v || !g_o || !d_q || !d_k || !d_v)))
    return da::fail(TTC_ERR_INVALID, "decay_attn_bwd: null pointer");
  const void* ops[3] = {q, k, v};
  for (int i = 0; i < 3; ++i)
    if (int rc = da::check_operand(ops[i], strides + 3 * i, 3, dtype)) return rc;
  const int64_t gs[3] = {T * H * dv, static_cast<int64_t>(H) * dv, dv};
  if (int rc = da::check_operand(g_o, gs, 0, dtype)) return rc;
  if (da::misaligned16(d_q) || da::misaligned16(d_k) || da::misaligned16(d_v))
    return da::fail(TTC_ERR_INVALID, "decay_attn_bwd: d_q, d_k and d_v must be 16-byte aligned");
  const da::Plan p = da::plan(T, n_seq, cu_seqlens != nullptr, H, dk, dv, 3, dtype);
  const int64_t sbytes = da::state_bytes(p, T, H, dk, dv, 3);
  const int grp = H / Hk;
  const int64_t rows = (cu_seqlens ? 1 : n_seq) * T;
  const int64_t need = sbytes + (grp > 1 ? 2 * rows * H * dk * 4 : 0);
  if (workspace_bytes < need || (need > 0 && (!workspace || da::misaligned16(workspace))))
    return da::fail(TTC_ERR_INVALID, "decay_attn_bwd: workspace missing, misaligned or smaller than ttc_decay_attn_workspace");
  if (T == 0 && d_initial_state == nullptr) return TTC_OK;
  da::Args A{};
  A.log_gamma = log_gamma;
  A.cu = cu_seqlens;
  A.T = T;
  A.n_seq = n_seq;
  A.H = H;
  A.seg_len = p.seg_len;
  A.n_seg = p.n_seg;
  A.items = p.items;
  A.parts = d_initial_state ? 3 : 2;
  char* ws = static_cast<char*>(workspace);
  float* part_q = grp > 1 ? reinterpret_cast<float*>(ws + sbytes) : nullptr;
  float* part_k = grp > 1 ? part_q + rows * H * dk : nullptr;
  const bool f32 = dtype == TTC_DTYPE_F32;
  da::Pass ps[3] = {};
  const auto set = [](int64_t* d, const int64_t* s) { d[0] = s[0], d[1] = s[1], d[2] = s[2]; };
  for (int i = 0; i < 3; ++i) {
    da::Pass& x = ps[i];
    x.seg = da::segmented(p, T) ? reinterpret_cast<float*>(ws) + i * (sbytes / 12) : nullptr;
    x.qg = x.kg = x.vg = 1;
    x.a = scale;
  }
  // dq: (g, v, k) forwards from S0^T
  da::Pass& dq = ps[0];
  dq.q = g_o, dq.k = v, dq.v = k, dq.vg = grp;
  set(dq.qs, gs), set(dq.ks, strides + 6), set(dq.vs, strides + 3);
  dq.o = grp > 1 ? static_cast<void*>(part_q) : d_q, dq.o_f32 = f32 || grp > 1;
  dq.init = initial_state, dq.isk = 1, dq.isv = dv;
  dq.kd = dv, dq.vd = dk, dq.b = scale, dq.u = 1.f;
  // dv: (k, q, g) backwards from dL/dS_T, whose last state is dL/dS0
  da::Pass& dvp = ps[1];
  dvp.q = k, dvp.k = q, dvp.v = g_o, dvp.qg = dvp.kg = grp;
  set(dvp.qs, strides + 3), set(dvp.ks, strides), set(dvp.vs, gs);
  dvp.o = d_v, dvp.o_f32 = f32;
  dvp.init = g_final_state, dvp.isk = dv, dvp.isv = 1, dvp.fin = d_initial_state;
  dvp.kd = dk, dvp.vd = dv, dvp.b = 1.f, dvp.u = scale, dvp.e = 1, dvp.reverse = 1;
  // dk: (v, g, q) backwards from (dL/dS_T)^T
  da::Pass& dkp = ps[2];
  dkp.q = v, dkp.k = g_o, dkp.v = q, dkp.vg = grp;
  set(dkp.qs, strides + 6), set(dkp.ks, gs), set(dkp.vs, strides);
  dkp.o = grp > 1 ? static_cast<void*>(part_k) : d_k, dkp.o_f32 = f32 || grp > 1;
  dkp.init = g_final_state, dkp.isk = 1, dkp.isv = dv;
  dkp.kd = dv, dkp.vd = dk, dkp.b = 1.f, dkp.u = scale, dkp.e = 1, dkp.reverse = 1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (int rc = da::run_passes(A, ps, 3, dtype, ps[0].seg != nullptr, status, st)) return rc;
  if (grp == 1 || rows == 0) return TTC_OK;
  const int64_t n4 = rows * Hk * dk / 4;
  const unsigned blocks = static_cast<unsigned>(std::min<int64_t>((n4 + 255) / 256, 148 * 16));
  if (f32)
    da::shared_heads_kernel<float><<<dim3(blocks, 2), 256, 0, st>>>(part_q, static_cast<float*>(d_q), part_k,
                                                                    static_cast<float*>(d_k), rows * Hk, grp, dk);
  else
    da::shared_heads_kernel<__nv_bfloat16><<<dim3(blocks, 2), 256, 0, st>>>(
        part_q, static_cast<__nv_bfloat16*>(d_q), part_k, static_cast<__nv_bfloat16*>(d_k), rows * Hk, grp, dk);
  return da::launched("shared_heads_kernel launch");
}

extern "C" int ttc_decay_attn_step(const void* q, const void* k, const void* v, const int64_t* strides,
                                   const float* log_gamma, float scale, float* state, int64_t slot_stride,
                                   const int* slots, int B, int n_slots, int H, int Hk, int dk, int dv, int dtype,
                                   void* o, void* stream) {
  if (int rc = da::check(1, B, false, H, Hk, dk, dv, dtype)) return rc;
  if (n_slots < 0 || (!slots && n_slots < B)) return da::fail(TTC_ERR_INVALID, "decay_attn_step: fewer states than rows");
  if (B == 0) return TTC_OK;
  if (!q || !k || !v || !strides || !log_gamma || !o || (n_slots > 0 && !state))
    return da::fail(TTC_ERR_INVALID, "decay_attn_step: null pointer");
  if (da::misaligned16(state) || slot_stride % 4 != 0)
    return da::fail(TTC_ERR_INVALID, "decay_attn_step: the states must start on 16-byte boundaries");
  // few rows: narrower column tiles, so that more CTAs share the states' bytes
  const int tile = static_cast<int64_t>(B) * H >= 296 || dv <= 32 ? dv : 32;
  const dim3 grid(B, H, (dv + tile - 1) / tile);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define TTC_STEP(T)                                                                                                   \
  da::decay_attn_step_kernel<T><<<grid, 256, 0, st>>>(                                                                \
      static_cast<const T*>(q), static_cast<const T*>(k), static_cast<const T*>(v), strides[0], strides[1], strides[2], \
      strides[3], strides[4], strides[5], log_gamma, scale, state, slot_stride, slots, B, n_slots, H, H / Hk, dk, dv,  \
      tile, static_cast<T*>(o))
  if (dtype == TTC_DTYPE_F32)
    TTC_STEP(float);
  else
    TTC_STEP(__nv_bfloat16);
#undef TTC_STEP
  return da::launched("decay_attn_step_kernel launch");
}
