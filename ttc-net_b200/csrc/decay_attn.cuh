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
// One CTA walks one segment of one (sequence, head, pass) with the transposed state S^T [dv x dk] in fp32
// registers over all blocks.  bf16: decay_attn_tc.cuh, on the 5th-generation tensor cores.  fp32:
// decay_attn_f32.cuh, on warp-level products of three bf16 parts each.
//
// A token's output does not depend on later tokens, whatever they hold: scores above the diagonal are set
// to 0, and where a block's values hold Inf or NaN (0 * NaN is NaN) the masked product runs term by term.
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
  int parts;  // bf16 only: parts of the decayed values in the state update
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
  if (A.n_seg == 1) {  // no sequence is cut: no search, which would cost a row of many sequences their square
    it.seq = x < A.n_seq ? x : -1;
    it.seg = 0;
    it.index = x;
    it.row0 = it.len = 0;
    if (it.seq >= 0) seq_range(A, it.seq, it.row0, it.len);
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
// 1 at n = 0.  A comparison, not fmaxf, which would make -1e4 of a NaN too.
__device__ __forceinline__ float decay_pow(float lg, int64_t n) {
  return static_cast<float>(exp(static_cast<double>(lg < -1e4f ? -1e4f : lg) * static_cast<double>(n)));
}

// Zeros in the rows behind the last packed sequence.  Over all heads they are one range of memory: each of the CTAs
// that a launch has for it (clearing_ctas for each head) takes an equal share of every stretch of it, 16 bytes a
// thread (vd is a multiple of 8 and the outputs start on 16-byte boundaries).  A row of 32 768 tokens, 32 heads of 128
// bf16, with 2 000 in use: the call takes 71 us; with one CTA a head, row after row, 4 840.
template <bool BF16>
__device__ __forceinline__ void zero_rows_behind(const Args& A, const Pass& P, int h, int tid, int threads) {
  int64_t row0, len;
  seq_range(A, A.n_seq - 1, row0, len);
  const int64_t bytes = static_cast<int64_t>(A.H) * P.vd * (BF16 && !P.o_f32 ? 2 : 4);
  uint4* const p = reinterpret_cast<uint4*>(static_cast<char*>(P.o) + (row0 + len) * bytes);
  const int64_t n = (A.T - row0 - len) * (bytes / 16);
  const int64_t share = static_cast<int64_t>(blockIdx.x - A.items) * A.H + h, shares = static_cast<int64_t>(gridDim.x - A.items) * A.H;
  for (int64_t i = share * threads + tid; i < n; i += shares * threads) p[i] = make_uint4(0u, 0u, 0u, 0u);
}

}  // namespace da
}  // namespace ttc
