// Attention with a fixed decay for each head, in blocks of 64 tokens.
//
//   S_t = gamma_h S_{t-1} + k_t^T v_t,   o_t = scale q_t S_t          (gamma_h = exp(log_gamma[h]))
//
// For a block of C = 64 tokens that starts from state S (i, j: places in the block):
//   o_i = a sum_{j <= i} gamma^{i-j} (q_i . k_j) v_j  +  b gamma^{i+1-e} q_i S
//   S'  = gamma^C S + u sum_j gamma^{C-1-j+e} k_j^T v_j
// Forward: a = b = scale, u = 1, e = 0.  The backward is the same recurrence three times
// (g = dL/do, R = dL/dS running backwards in time from the last state's gradient):
//   dq = this with (q, k, v) := (g, v, k), start S0^T
//   dv = this backwards in time with (k, q, g), start dL/dS_T,   a = scale, b = 1, u = scale, e = 1
//   dk = this backwards in time with (v, g, q), start (dL/dS_T)^T, the same factors; the last
//        state of the dv pass is dL/dS0.
//
// One CTA walks one segment of one (sequence, head): DV / 16 warps, warp w owns rows 16w..16w+15
// of the transposed state S^T [DV x DK], which stays in its fp32 accumulators over all blocks.
// The accumulator layout of S^T is the layout of an A operand, so q S is formed as
// o^T = S^T q^T without the state ever leaving the registers; the update accumulates
// S^T += (u gamma^.. v)^T k in place.  The 64 x 64 scores go through shared memory once.
//
// Roundings (bf16 inputs, NP = 1): scores and the copy of S that multiplies q are rounded to
// bf16 (each adds an error of the size of the output's own rounding); the decayed values of the
// state update are two or three bf16 parts (16 or 24 bits; three where the last state is an
// output), so that the state itself is right to fp32.  fp32 inputs (NP = 3): every operand is three bf16
// parts and the products whose parts' ranks add up to at most 2 are formed (6 of 9), which
// leaves out terms of 2^-24.  tf32 in three products would cost the same time and drop 2^-22.
// The tensor core's fp32 sums cut instead of rounding, a bias that grows with the number of
// additions: the products of the first parts and the small corrections have accumulators of their own,
// and a block's sum is formed from zero and added to the state by an ordinary rounded fma
// (accumulating in place put 3e-6 on the state of 3000 tokens, this way it is under 1e-6).
//
// A token's output does not depend on later tokens, whatever they hold: scores above the
// diagonal are set to 0, and where a block's values hold Inf or NaN (0 * NaN is NaN) the
// masked product runs term by term instead (`slow_pv`).
#pragma once

#include <cuda_runtime.h>

#include "lqr_common.cuh"
#include "mma_bf16.cuh"

namespace ttc {
namespace da {

constexpr int C = 64;  // tokens of a block

// One recurrence; every stride in elements.  `grp`: heads that share one head of the operand.
struct Pass {
  const void *q, *k, *v;
  int64_t qs[3], ks[3], vs[3];  // batch, token, head
  int qg, kg, vg;
  void* o;  // [B, T, H, vd] contiguous
  int o_f32;
  const float* init;  // may be null; element (n, h, kr, vr) at ((n H + h) kd vd + kr isk + vr isv)
  int64_t isk, isv;
  float* fin;  // may be null, [n, H, kd, vd] contiguous
  float* seg;  // states at the segments' starts [items, H, kd, vd], null when one segment is all
  int kd, vd;
  float a, b, u;
  int e, reverse;
};

struct Args {
  Pass pass[3];
  const float* log_gamma;
  const int* cu;  // null: B sequences of T tokens
  int64_t T;      // tokens of a sequence, or of the packed row
  int n_seq, H, seg_len, n_seg;
  int items;  // upper bound on the number of (sequence, segment) pairs
  int parts;  // bf16 parts of the decayed values in the state update (NP = 1)
};

struct Item {
  int seq, seg;       // seq < 0: nothing to do
  int64_t row0, len;  // first row and length of the sequence
  int64_t index;      // of the first segment
};

// Sequence n of the packed row.  Bad offsets (decreasing, past the end) are cut to the row.
__device__ __forceinline__ void seq_range(const Args& A, int n, int64_t& row0, int64_t& len) {
  if (A.cu == nullptr) {
    row0 = 0;
    len = A.T;
    return;
  }
  const int64_t s = A.cu[n], e = A.cu[n + 1];
  row0 = s < 0 ? 0 : (s > A.T ? A.T : s);
  const int64_t end = e < row0 ? row0 : (e > A.T ? A.T : e);
  len = end - row0;
}

__device__ __forceinline__ int segs_of(const Args& A, int64_t len) {
  const int64_t s = (len + A.seg_len - 1) / A.seg_len;
  return s < 1 ? 1 : static_cast<int>(s);
}

// The (sequence, segment) pair number x; executed by whole warps, all lanes get the result.
__device__ __forceinline__ Item find_item(const Args& A, int x) {
  Item it;
  if (A.cu == nullptr) {
    it.seq = x / A.n_seg;
    it.seg = x - it.seq * A.n_seg;
    it.index = static_cast<int64_t>(it.seq) * A.n_seg;
    if (it.seq >= A.n_seq) it.seq = -1;
    it.row0 = 0;
    it.len = A.T;
    return it;
  }
  const int lane = threadIdx.x & 31;
  int64_t before = 0;
  for (int n0 = 0; n0 < A.n_seq; n0 += 32) {
    const int n = n0 + lane;
    int64_t row0 = 0, len = 0;
    int cnt = 0;
    if (n < A.n_seq) {
      seq_range(A, n, row0, len);
      cnt = segs_of(A, len);
    }
    int sum = cnt;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += y;
    }
    const bool mine = n < A.n_seq && x >= before + sum - cnt && x < before + sum;
    const unsigned who = __ballot_sync(0xffffffffu, mine);
    if (who) {
      const int src = __ffs(who) - 1;
      it.seq = n0 + src;
      const int first = __shfl_sync(0xffffffffu, sum - cnt, src);
      it.index = before + first;
      it.seg = static_cast<int>(x - it.index);
      it.row0 = __shfl_sync(0xffffffffu, row0, src);
      it.len = __shfl_sync(0xffffffffu, len, src);
      return it;
    }
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
  it.seq = -1;
  it.seg = 0;
  it.row0 = it.len = it.index = 0;
  return it;
}

// gamma^n; log gamma = -inf (no memory) is taken as -1e4, whose powers are 0 from n = 1 on and
// 1 at n = 0.
__device__ __forceinline__ float decay_pow(float lg, int64_t n) {
  return static_cast<float>(exp(static_cast<double>(fmaxf(lg, -1e4f)) * static_cast<double>(n)));
}

// Rows r of a block (token t0 + r of the segment's sequence) into a swizzled tile; rows past the
// block's end and columns past `d` are zeros.
template <int COLS, int NP, int THREADS>
__device__ __forceinline__ void load_tile(uint32_t dst, const void* src, int64_t row_stride, int64_t first, int64_t step,
                                          int rows, int d) {
  constexpr int PIECES = COLS / 8;
  for (int x = threadIdx.x; x < C * PIECES; x += THREADS) {
    const int r = x / PIECES, c = x % PIECES;
    const bool on = r < rows && c * 8 < d;
    const int64_t off = on ? (first + step * r) * row_stride + c * 8 : 0;
    const uint32_t at = dst + mma::tile_off<COLS>(r, c);
    if constexpr (NP == 1) {
      mma::cp16(at, static_cast<const __nv_bfloat16*>(src) + off, on ? 16 : 0);
    } else {
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
      if (on) {
        const float* p = static_cast<const float*>(src) + off;
        a = *reinterpret_cast<const float4*>(p);
        b = *reinterpret_cast<const float4*>(p + 4);
      }
      uint32_t w[4][NP];
      mma::split2<NP>(a.x, a.y, w[0]);
      mma::split2<NP>(a.z, a.w, w[1]);
      mma::split2<NP>(b.x, b.y, w[2]);
      mma::split2<NP>(b.z, b.w, w[3]);
#pragma unroll
      for (int s = 0; s < NP; ++s)
        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at + s * (C * COLS * 2)), "r"(w[0][s]), "r"(w[1][s]),
                     "r"(w[2][s]), "r"(w[3][s])
                     : "memory");
    }
  }
}

template <int DK, int DV, int NP, bool STATE_ONLY>
struct Shape {
  static constexpr int WARPS = DV / 16, THREADS = 32 * WARPS;
  static constexpr int STAGES = NP == 1 ? 2 : 1;
  static constexpr int QB = STATE_ONLY ? 0 : C * DK * 2 * NP;
  static constexpr int KB = C * DK * 2 * NP, VB = C * DV * 2 * NP;
  static constexpr int STAGE = QB + KB + VB;
  static constexpr int PB = STATE_ONLY ? 0 : C * C * 2 * NP;
  static constexpr int TABLE = 80 * 4;  // gamma^0 .. gamma^64
  static constexpr int SMEM = STAGES * STAGE + PB + TABLE;
};

template <int NP>
__device__ __forceinline__ float tile_value(const char* tile, uint32_t off, int plane_bytes) {
  float v = 0.f;
#pragma unroll
  for (int s = NP - 1; s >= 0; --s)
    v += __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(tile + off + s * plane_bytes));
  return v;
}

// The rows and tokens of one warp's product of scores and values, term by term and only over
// j <= i, for blocks whose values are not all finite.
template <int DV, int NP>
__device__ __noinline__ void slow_pv(float (&acc)[4][4], const char* Ps, const char* Vs, int half, int row) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int nt = 0; nt < 4; ++nt)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int i = 32 * half + 8 * nt + 2 * t + (x & 1), r = row + g + 8 * (x >> 1);
      float s = 0.f;
      for (int j = 0; j <= i; ++j)
        s = fmaf(tile_value<NP>(Ps, mma::tile_off<C>(i, j >> 3) + (j & 7) * 2, C * C * 2),
                 tile_value<NP>(Vs, mma::tile_off<DV>(j, r >> 3) + (r & 7) * 2, C * DV * 2), s);
      acc[nt][x] += s;
    }
}

// Zeros in the rows behind the last packed sequence.
template <bool BF16>
__device__ __forceinline__ void zero_rows_behind(const Args& A, const Pass& P, int h, int tid, int threads) {
  int64_t row0, len;
  seq_range(A, A.n_seq - 1, row0, len);
  for (int64_t r = row0 + len; r < A.T; ++r)
    for (int c = tid; c < P.vd; c += threads) {
      const int64_t at = (r * A.H + h) * P.vd + c;
      if (BF16 && !P.o_f32)
        static_cast<__nv_bfloat16*>(P.o)[at] = __float2bfloat16_rn(0.f);
      else
        static_cast<float*>(P.o)[at] = 0.f;
    }
}

// STATE_ONLY: the sums u gamma^.. k^T v of the segments alone, from a zero state.
template <int DK, int DV, int NP, bool STATE_ONLY>
__global__ void __launch_bounds__(Shape<DK, DV, NP, STATE_ONLY>::THREADS) decay_attn_kernel(const __grid_constant__ Args A) {
  using S = Shape<DK, DV, NP, STATE_ONLY>;
  constexpr int NA = NP == 1 ? 1 : 2;  // accumulators: first parts' products, the others'
  extern __shared__ __align__(128) char smem[];
  const Pass& P = A.pass[blockIdx.z];
  const int h = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  char* const Ps = smem + S::STAGES * S::STAGE;
  float* const pw = reinterpret_cast<float*>(Ps + S::PB);

  if (!STATE_ONLY && A.cu != nullptr && static_cast<int>(blockIdx.x) == A.items) {
    zero_rows_behind<NP == 1>(A, P, h, tid, S::THREADS);
    return;
  }
  const Item it = find_item(A, blockIdx.x);
  if (it.seq < 0) return;
  const int64_t s0 = static_cast<int64_t>(it.seg) * A.seg_len;
  const int64_t left = it.len - s0;
  const int seg_rows = static_cast<int>(left < A.seg_len ? (left > 0 ? left : 0) : A.seg_len);
  const int blocks = (seg_rows + C - 1) / C;
  const bool last_seg = s0 + seg_rows >= it.len;
  // the scan over the segments needs no sum behind the last one unless the last state is wanted
  if (STATE_ONLY && last_seg && P.fin == nullptr) return;

  const int bi = A.cu == nullptr ? it.seq : 0;
  const int64_t es = NP == 1 ? 2 : 4;
  const char* qb = static_cast<const char*>(P.q) + (bi * P.qs[0] + (h / P.qg) * P.qs[2]) * es;
  const char* kb = static_cast<const char*>(P.k) + (bi * P.ks[0] + (h / P.kg) * P.ks[2]) * es;
  const char* vb = static_cast<const char*>(P.v) + (bi * P.vs[0] + (h / P.vg) * P.vs[2]) * es;
  const int64_t step = P.reverse ? -1 : 1;
  const int64_t first = it.row0 + (P.reverse ? it.len - 1 - s0 : s0);  // row of the segment's first token

  auto load_block = [&](int c) {
    const int rows = min(C, seg_rows - c * C);
    const uint32_t st = mma::smem_u32(smem + (c % S::STAGES) * S::STAGE);
    const int64_t f = first + step * c * C;
    if constexpr (!STATE_ONLY) load_tile<DK, NP, S::THREADS>(st, qb, P.qs[1], f, step, rows, P.kd);
    load_tile<DK, NP, S::THREADS>(st + S::QB, kb, P.ks[1], f, step, rows, P.kd);
    load_tile<DV, NP, S::THREADS>(st + S::QB + S::KB, vb, P.vs[1], f, step, rows, P.vd);
    mma::cp_commit();
  };
  if (S::STAGES == 2 && blocks > 0) load_block(0);

  if (tid <= C) pw[tid] = decay_pow(A.log_gamma[h], tid);
  if (S::THREADS < C + 1)
    for (int i = tid + S::THREADS; i <= C; i += S::THREADS) pw[i] = decay_pow(A.log_gamma[h], i);

  // S^T: rows 16 warp + g (+8), columns 8 n + 2t (+1)
  float st[DK / 8][4];
  const int row = 16 * warp;
  const int64_t sbase = (static_cast<int64_t>(it.seq) * A.H + h) * P.kd * P.vd;
  const int64_t gbase = ((it.index + it.seg) * A.H + h) * P.kd * P.vd;
  const float* src = nullptr;
  int64_t sk = P.vd, sv = 1;
  if (!STATE_ONLY) {
    if (P.seg != nullptr) {
      src = P.seg + gbase;
    } else if (P.init != nullptr) {
      src = P.init + sbase;
      sk = P.isk;
      sv = P.isv;
    }
  }
#pragma unroll
  for (int n = 0; n < DK / 8; ++n)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int kr = 8 * n + 2 * t + (x & 1), vr = row + g + 8 * (x >> 1);
      st[n][x] = src != nullptr && kr < P.kd && vr < P.vd ? src[kr * sk + vr * sv] : 0.f;
    }
  bool zero_state = src == nullptr;

  // lane addresses of the four ldmatrix forms (rows, pieces inside a 16 x 16 corner)
  const int m = lane >> 3, r8 = lane & 7;

  for (int c = 0; c < blocks; ++c) {
    const int rows = min(C, seg_rows - c * C);
    if (S::STAGES == 1) {
      if (c > 0) __syncthreads();  // the tiles are read by the block before
      load_block(c);
    }
    mma::cp_wait<0>();
    __syncthreads();
    if (S::STAGES == 2 && c + 1 < blocks) load_block(c + 1);
    const char* const base = smem + (c % S::STAGES) * S::STAGE;
    const uint32_t Qs = mma::smem_u32(base), Ks = Qs + S::QB, Vs = Ks + S::KB, Pa = mma::smem_u32(Ps);
    const char* const Vc = base + S::QB + S::KB;

    if constexpr (!STATE_ONLY) {
      // scores: jobs (16 rows b, half of the b's 2b + 2 column tiles), given out so that every
      // warp has the same number of tiles where there are fewer than 8 warps
      auto job = [&](int b, int half) {
        const int nt0 = half ? b + 1 : 0;
        float acc[NA][4][4] = {};
#pragma unroll
        for (int ks = 0; ks < DK / 32; ++ks) {
          uint32_t a[NP][2][4];
#pragma unroll
          for (int s = 0; s < NP; ++s)
#pragma unroll
            for (int k2 = 0; k2 < 2; ++k2)
              mma::ldsm4(a[s][k2], Qs + s * (C * DK * 2) +
                                       mma::tile_off<DK>(16 * b + (m & 1) * 8 + r8, ks * 4 + k2 * 2 + (m >> 1)));
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            if (n <= b) {
              uint32_t bf[NP][4];
#pragma unroll
              for (int s = 0; s < NP; ++s)
                mma::ldsm4(bf[s], Ks + s * (C * DK * 2) + mma::tile_off<DK>(8 * (nt0 + n) + r8, ks * 4 + m));
#pragma unroll
              for (int sa = NP - 1; sa >= 0; --sa)
#pragma unroll
                for (int sb = NP - 1 - sa; sb >= 0; --sb) {
                  mma::mma16816(acc[sa + sb ? NA - 1 : 0][n], a[sa][0], bf[sb][0], bf[sb][1]);
                  mma::mma16816(acc[sa + sb ? NA - 1 : 0][n], a[sa][1], bf[sb][2], bf[sb][3]);
                }
            }
          }
        }
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          if (n <= b) {
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const int i = 16 * b + g + 8 * y, j = 8 * (nt0 + n) + 2 * t;
              float v0 = acc[0][n][2 * y], v1 = acc[0][n][2 * y + 1];
              if (NA == 2) v0 += acc[NA - 1][n][2 * y], v1 += acc[NA - 1][n][2 * y + 1];
              v0 = j <= i ? v0 * (P.a * pw[i - j]) : 0.f;
              v1 = j + 1 <= i ? v1 * (P.a * pw[i - j - 1]) : 0.f;
              uint32_t w[NP];
              mma::split2<NP>(v0, v1, w);
#pragma unroll
              for (int s = 0; s < NP; ++s)
                *reinterpret_cast<uint32_t*>(Ps + s * (C * C * 2) + mma::tile_off<C>(i, nt0 + n) + t * 4) = w[s];
            }
          }
        }
      };
      if constexpr (S::WARPS == 8) {
        job(warp & 3, warp >> 2);
      } else if constexpr (S::WARPS == 4) {
        job(warp >> 1, warp & 1);
        job(3 - (warp >> 1), warp & 1);
      } else {
#pragma unroll 1
        for (int b = 0; b < 4; ++b) job(b, warp);
      }
      __syncthreads();
    }

    // values with Inf or NaN in this warp's rows?
    bool odd = false;
    if constexpr (!STATE_ONLY) {
      float chk = 0.f;
#pragma unroll
      for (int kb16 = 0; kb16 < 4; ++kb16) {
        uint32_t a[4];
        mma::ldsm4t(a, Vs + mma::tile_off<DV>(16 * kb16 + (m >> 1) * 8 + r8, row / 8 + (m & 1)));
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          chk = fmaf(mma::lo_f(a[x]), 0.f, chk);
          chk = fmaf(mma::hi_f(a[x]), 0.f, chk);
        }
      }
      odd = __any_sync(0xffffffffu, chk != 0.f || chk != chk);

#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (32 * half < rows) {
          float acc[NA][4][4] = {};
          if (!zero_state) {
#pragma unroll
            for (int ks = 0; ks < DK / 16; ++ks) {
              uint32_t a[NP][4];
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                uint32_t w[NP];
                mma::split2<NP>(st[2 * ks + (y >> 1)][2 * (y & 1)], st[2 * ks + (y >> 1)][2 * (y & 1) + 1], w);
#pragma unroll
                for (int s = 0; s < NP; ++s) a[s][y] = w[s];
              }
#pragma unroll
              for (int n2 = 0; n2 < 2; ++n2) {
                uint32_t bf[NP][4];
#pragma unroll
                for (int s = 0; s < NP; ++s)
                  mma::ldsm4(bf[s], Qs + s * (C * DK * 2) +
                                        mma::tile_off<DK>(32 * half + 16 * n2 + (m >> 1) * 8 + r8, 2 * ks + (m & 1)));
#pragma unroll
                for (int sa = NP - 1; sa >= 0; --sa)
#pragma unroll
                  for (int sb = NP - 1 - sa; sb >= 0; --sb) {
                    mma::mma16816(acc[sa + sb ? NA - 1 : 0][2 * n2], a[sa], bf[sb][0], bf[sb][1]);
                    mma::mma16816(acc[sa + sb ? NA - 1 : 0][2 * n2 + 1], a[sa], bf[sb][2], bf[sb][3]);
                  }
              }
            }
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
              for (int y = 0; y < 2; ++y) {
                const float f = P.b * pw[32 * half + 8 * n + 2 * t + y + 1 - P.e];
#pragma unroll
                for (int w = 0; w < NA; ++w) {
                  acc[w][n][y] *= f;
                  acc[w][n][y + 2] *= f;
                }
              }
          }
          if (!odd) {
#pragma unroll
            for (int kb16 = 0; kb16 < 4; ++kb16) {
              if (kb16 < 2 + 2 * half) {
                uint32_t a[NP][4];
#pragma unroll
                for (int s = 0; s < NP; ++s)
                  mma::ldsm4t(a[s], Vs + s * (C * DV * 2) +
                                        mma::tile_off<DV>(16 * kb16 + (m >> 1) * 8 + r8, row / 8 + (m & 1)));
#pragma unroll
                for (int n2 = 0; n2 < 2; ++n2) {
                  if (kb16 <= 2 * half + n2) {  // token tiles 16 (2 half + n2): scores beyond are 0
                    uint32_t bf[NP][4];
#pragma unroll
                    for (int s = 0; s < NP; ++s)
                      mma::ldsm4(bf[s], Pa + s * (C * C * 2) +
                                            mma::tile_off<C>(32 * half + 16 * n2 + (m >> 1) * 8 + r8, 2 * kb16 + (m & 1)));
#pragma unroll
                    for (int sa = NP - 1; sa >= 0; --sa)
#pragma unroll
                      for (int sb = NP - 1 - sa; sb >= 0; --sb) {
                        mma::mma16816(acc[sa + sb ? NA - 1 : 0][2 * n2], a[sa], bf[sb][0], bf[sb][1]);
                        mma::mma16816(acc[sa + sb ? NA - 1 : 0][2 * n2 + 1], a[sa], bf[sb][2], bf[sb][3]);
                      }
                  }
                }
              }
            }
          } else {
            slow_pv<DV, NP>(acc[0], Ps, Vc, half, row);
          }
          if (NA == 2) {
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
              for (int x = 0; x < 4; ++x) acc[0][n][x] += acc[NA - 1][n][x];
          }
          // o^T -> o: element (token 2t, 2t+1; value row g, g + 8)
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const int i0 = 32 * half + 8 * n;
            if (NP == 1 && !P.o_f32) {
#pragma unroll
              for (int y = 0; y < 2; ++y) {
                const uint32_t w = mma::transpose8(mma::pack2(acc[0][n][2 * y], acc[0][n][2 * y + 1]));
                const int i = i0 + g, vr = row + 8 * y + 2 * t;
                if (i < rows && vr < P.vd) {
                  const int64_t tok = bi * A.T + first + step * (c * C + i);
                  *reinterpret_cast<uint32_t*>(static_cast<__nv_bfloat16*>(P.o) + (tok * A.H + h) * P.vd + vr) = w;
                }
              }
            } else {
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                const int i = i0 + 2 * t + (x & 1), vr = row + g + 8 * (x >> 1);
                if (i < rows && vr < P.vd) {
                  const int64_t tok = bi * A.T + first + step * (c * C + i);
                  static_cast<float*>(P.o)[(tok * A.H + h) * P.vd + vr] = acc[0][n][x];
                }
              }
            }
          }
        }
      }
    }

    // the state behind this block
    if (STATE_ONLY || c + 1 < blocks || (P.seg == nullptr && P.fin != nullptr)) {
      const float keep = pw[rows];
      const bool three = NP == 3 || A.parts == 3;
#pragma unroll
      for (int p2 = 0; p2 < 2; ++p2) {  // tokens 0..31 and 32..63
        if (32 * p2 < rows) {
          uint32_t a[2][3][4];
#pragma unroll
          for (int q2 = 0; q2 < 2; ++q2) {
            const int kb16 = 2 * p2 + q2;
            float va[4][2] = {};
#pragma unroll
            for (int s = NP - 1; s >= 0; --s) {
              uint32_t w[4];
              mma::ldsm4t(w, Vs + s * (C * DV * 2) + mma::tile_off<DV>(16 * kb16 + (m >> 1) * 8 + r8, row / 8 + (m & 1)));
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                va[y][0] += mma::lo_f(w[y]);
                va[y][1] += mma::hi_f(w[y]);
              }
            }
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const int j = 16 * kb16 + 8 * (y >> 1) + 2 * t;
              const float f0 = j < rows ? P.u * pw[rows - 1 - j + P.e] : 0.f;
              const float f1 = j + 1 < rows ? P.u * pw[rows - 2 - j + P.e] : 0.f;
              uint32_t w[3];
              mma::split2<3>(va[y][0] * f0, va[y][1] * f1, w);
              a[q2][0][y] = w[0];
              a[q2][1][y] = w[1];
              a[q2][2][y] = w[2];
            }
          }
#pragma unroll
          for (int n2 = 0; n2 < DK / 16; ++n2) {
            float add[2][2][4] = {};  // first parts' products; the others'
#pragma unroll
            for (int q2 = 0; q2 < 2; ++q2) {
              uint32_t bf[NP][4];
#pragma unroll
              for (int s = 0; s < NP; ++s)
                mma::ldsm4t(bf[s], Ks + s * (C * DK * 2) +
                                       mma::tile_off<DK>(32 * p2 + 16 * q2 + (m & 1) * 8 + r8, 2 * n2 + (m >> 1)));
#pragma unroll
              for (int sb = 0; sb < NP; ++sb)
#pragma unroll
                for (int sa = 2 - sb; sa >= 0; --sa)
                  if (sa < 2 || three) {
                    mma::mma16816(add[sa + sb > 0][0], a[q2][sa], bf[sb][0], bf[sb][1]);
                    mma::mma16816(add[sa + sb > 0][1], a[q2][sa], bf[sb][2], bf[sb][3]);
                  }
            }
#pragma unroll
            for (int y = 0; y < 2; ++y)
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                const float d = add[0][y][x] + add[1][y][x];
                st[2 * n2 + y][x] = p2 == 0 ? fmaf(keep, st[2 * n2 + y][x], d) : st[2 * n2 + y][x] + d;
              }
          }
        }
      }
      zero_state = false;
    }
  }

  float* dst = nullptr;
  if (STATE_ONLY)
    dst = P.seg + gbase;
  else if (P.seg == nullptr && P.fin != nullptr)
    dst = P.fin + sbase;
  if (dst != nullptr) {
#pragma unroll
    for (int n = 0; n < DK / 8; ++n)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int kr = 8 * n + 2 * t + (x & 1), vr = row + g + 8 * (x >> 1);
        if (kr < P.kd && vr < P.vd) dst[static_cast<int64_t>(kr) * P.vd + vr] = st[n][x];
      }
  }
}

}  // namespace da
}  // namespace ttc
