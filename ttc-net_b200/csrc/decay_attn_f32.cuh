// The recurrence of decay_attn.cuh for fp32 on warp-level bf16 products.
//
// Every fp32 operand is three bf16 parts (24 bits), and the six products whose parts' ranks add up to at most 2
// are formed, which leaves out terms of 2^-24; tf32 in three products would cost the same time and drop 2^-22.
// The tensor core's fp32 sums cut instead of rounding, a bias that grows with the number of additions: the products of
// the first parts and the small corrections have accumulators of their own, and a block's sum is formed from
// zero and added to the state by an ordinary rounded fma (accumulating in place put 3e-6 on the state of 3000
// tokens, this way it is under 2e-7).
//
// Eight warps.  Warp (rg, tg) owns rows 16 rg .. 16 rg + 15 of S^T, all of them for each of the 8 / (DV / 16)
// token groups tg: the layout of its accumulators is the layout of an A operand, so o^T = S^T q^T is formed for the
// group's tokens without the state leaving the registers, at the price of updating it once a group.  The parts of
// q, k, v and of the 64 x 64 scores lie in shared memory; the next block's values are on their way in registers
// meanwhile where they are few enough (2 DK + DV <= 192).  Heads of at most 32 x 32 fit twice on an SM.
// Bound by issuing and waiting: two warps to a scheduler, the tensor pipe 29 % busy with the six products at 32 x 64.
// 4 x 1001 tokens, 16 heads of 32 / 64: forward 86 us, backward 238; 8 x 1024, 37 heads of 64: 298 and 885.
#pragma once

#include "decay_attn.cuh"

namespace ttc {
namespace da {

constexpr int NP = 3;  // parts
constexpr int kF32Threads = 256;

// This thread's share of a [64 x COLS] tile on its way to shared memory, 8 values a piece.
template <int COLS>
struct TileRegs {
  static constexpr int PIECES = COLS / 8, N = C * PIECES / kF32Threads;
  float4 v[N][2];
  // rows r of a block (token first + step r); rows past the block's end and columns past d are zeros
  __device__ __forceinline__ void load(const float* src, int64_t row_stride, int64_t first, int64_t step, int rows, int d) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int x = threadIdx.x + kF32Threads * i, r = x / PIECES, c = x % PIECES;
      v[i][0] = v[i][1] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < rows && c * 8 < d) {
        const float4* p = reinterpret_cast<const float4*>(src + (first + step * r) * row_stride + c * 8);
        v[i][0] = p[0];
        v[i][1] = p[1];
      }
    }
  }
  __device__ __forceinline__ void store(uint32_t dst) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int x = threadIdx.x + kF32Threads * i, r = x / PIECES, c = x % PIECES;
      uint32_t w[4][NP];
      mma::split2<NP>(v[i][0].x, v[i][0].y, w[0]);
      mma::split2<NP>(v[i][0].z, v[i][0].w, w[1]);
      mma::split2<NP>(v[i][1].x, v[i][1].y, w[2]);
      mma::split2<NP>(v[i][1].z, v[i][1].w, w[3]);
#pragma unroll
      for (int s = 0; s < NP; ++s)
        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst + mma::tile_off<COLS>(r, c) + s * (C * COLS * 2)),
                     "r"(w[0][s]), "r"(w[1][s]), "r"(w[2][s]), "r"(w[3][s])
                     : "memory");
    }
  }
};

template <int DK, int DV, bool STATE_ONLY>
struct F32Shape {
  static constexpr int RG = DV / 16, TG = 8 / RG;
  static constexpr int QB = STATE_ONLY ? 0 : C * DK * 2 * NP, KB = C * DK * 2 * NP, VB = C * DV * 2 * NP;
  static constexpr int PB = STATE_ONLY ? 0 : C * C * 2 * NP;
  static constexpr int TABLE = 80 * 4;  // gamma^0 .. gamma^64
  static constexpr int SMEM = QB + KB + VB + PB + TABLE;
  static constexpr bool AHEAD = (STATE_ONLY ? DK : 2 * DK) + DV <= 192;
  // the sums alone: a token group has its own columns of S^T instead, 16 at least
  static constexpr int CG = STATE_ONLY ? (TG < DK / 16 ? TG : DK / 16) : 1;
  static constexpr int N2 = DK / 16 / CG;  // 16-column pieces of S^T of a warp
};

__device__ __forceinline__ float tile_value(const char* tile, uint32_t off, int plane_bytes) {
  float v = 0.f;
#pragma unroll
  for (int s = NP - 1; s >= 0; --s)
    v += __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(tile + off + s * plane_bytes));
  return v;
}

// A warp's product of scores and values for 8 NT tokens from i0 on, term by term and only over j <= i, for
// blocks whose values are not all finite.
template <int DV, int NT>
__device__ __noinline__ void slow_pv(float (&out)[NT][4], const char* Ps, const char* Vs, int i0, int row) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int i = i0 + 8 * nt + 2 * t + (x & 1), r = row + g + 8 * (x >> 1);
      float s = 0.f;
#pragma unroll 1
      for (int j = 0; j <= i; ++j)
        s = fmaf(tile_value(Ps, mma::tile_off<C>(i, j >> 3) + (j & 7) * 2, C * C * 2),
                 tile_value(Vs, mma::tile_off<DV>(j, r >> 3) + (r & 7) * 2, C * DV * 2), s);
      out[nt][x] = s;
    }
}

// STATE_ONLY: the sums u gamma^.. k^T v of the segments alone, from a zero state.
template <int DK, int DV, bool STATE_ONLY>
__global__ void __launch_bounds__(kF32Threads, (DK + DV <= 64 ? 2 : 1)) decay_attn_f32_kernel(const __grid_constant__ Args A) {
  using S = F32Shape<DK, DV, STATE_ONLY>;
  extern __shared__ __align__(128) char smem[];
  const Pass& P = A.pass[blockIdx.z];
  const int h = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int rg = warp % S::RG, tg = warp / S::RG;
  char* const Ps = smem + S::QB + S::KB + S::VB;
  float* const pw = reinterpret_cast<float*>(Ps + S::PB);

  if (!STATE_ONLY && A.cu != nullptr && static_cast<int>(blockIdx.x) >= A.items) {
    zero_rows_behind<false>(A, P, h, tid, kF32Threads);
    return;
  }
  const Item it = find_item(A, blockIdx.x);
  if (it.seq < 0) return;
  const int64_t s0 = static_cast<int64_t>(it.seg) * A.seg_len;
  const int64_t left = it.len - s0;
  const int seg_rows = static_cast<int>(left < A.seg_len ? (left > 0 ? left : 0) : A.seg_len);
  const int blocks = (seg_rows + C - 1) / C;
  // the scan over the segments needs no sum behind the last one unless the last state is wanted
  if (STATE_ONLY && s0 + seg_rows >= it.len && P.fin == nullptr) return;

  const int bi = A.cu == nullptr ? it.seq : 0;
  const float* qb = static_cast<const float*>(P.q) + bi * P.qs[0] + (h / P.qg) * P.qs[2];
  const float* kb = static_cast<const float*>(P.k) + bi * P.ks[0] + (h / P.kg) * P.ks[2];
  const float* vb = static_cast<const float*>(P.v) + bi * P.vs[0] + (h / P.vg) * P.vs[2];
  const int64_t step = P.reverse ? -1 : 1;
  const int64_t first = it.row0 + (P.reverse ? it.len - 1 - s0 : s0);  // row of the segment's first token

  const uint32_t Qs = mma::smem_u32(smem), Ks = Qs + S::QB, Vs = Ks + S::KB, Pa = mma::smem_u32(Ps);
  const char* const Vc = smem + S::QB + S::KB;
  TileRegs<DK> rq, rk;
  TileRegs<DV> rv;
  auto load_q = [&](int c) { rq.load(qb, P.qs[1], first + step * c * C, step, min(C, seg_rows - c * C), P.kd); };
  auto load_k = [&](int c) { rk.load(kb, P.ks[1], first + step * c * C, step, min(C, seg_rows - c * C), P.kd); };
  auto load_v = [&](int c) { rv.load(vb, P.vs[1], first + step * c * C, step, min(C, seg_rows - c * C), P.vd); };
  if (S::AHEAD && blocks > 0) {
    if (!STATE_ONLY) load_q(0);
    load_k(0);
    load_v(0);
  }
  if (tid <= C) pw[tid] = decay_pow(A.log_gamma[h], tid);

  // S^T: rows 16 rg + g (+8), columns col0 + 8 n + 2t (+1)
  float st[2 * S::N2][4];
  const int row = 16 * rg, col0 = STATE_ONLY ? tg * 16 * S::N2 : 0;
  const bool owner = STATE_ONLY ? tg < S::CG : true;
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
  for (int n = 0; n < 2 * S::N2; ++n)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int kr = col0 + 8 * n + 2 * t + (x & 1), vr = row + g + 8 * (x >> 1);
      st[n][x] = src != nullptr && kr < P.kd && vr < P.vd ? src[kr * sk + vr * sv] : 0.f;
    }
  bool zero_state = src == nullptr;

  const int m = lane >> 3, r8 = lane & 7;  // lane's matrix and row in ldmatrix

#pragma unroll 1
  for (int c = 0; c < blocks; ++c) {
    const int rows = min(C, seg_rows - c * C);
    if (c > 0) __syncthreads();  // the tiles are read by the block before
    if (S::AHEAD) {
      if (!STATE_ONLY) rq.store(Qs);
      rk.store(Ks);
      rv.store(Vs);
      if (c + 1 < blocks) {
        if (!STATE_ONLY) load_q(c + 1);
        load_k(c + 1);
        load_v(c + 1);
      }
    } else {
      if (!STATE_ONLY) {
        load_q(c);
        rq.store(Qs);
      }
      load_k(c);
      rk.store(Ks);
      load_v(c);
      rv.store(Vs);
    }
    __syncthreads();

    if constexpr (!STATE_ONLY) {
      {  // scores: warp (b, half) has 16 rows b and half of their 2b + 2 column tiles
        const int b = warp & 3, nt0 = (warp >> 2) ? b + 1 : 0;
        float acc[2][4][4] = {};
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
                  mma::mma16816(acc[sa + sb > 0][n], a[sa][0], bf[sb][0], bf[sb][1]);
                  mma::mma16816(acc[sa + sb > 0][n], a[sa][1], bf[sb][2], bf[sb][3]);
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
              float v0 = acc[0][n][2 * y] + acc[1][n][2 * y], v1 = acc[0][n][2 * y + 1] + acc[1][n][2 * y + 1];
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
      }
      __syncthreads();

      // values with Inf or NaN in this warp's rows?
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
      const bool odd = __any_sync(0xffffffffu, chk != 0.f || chk != chk);

      // this warp's groups of 16 tokens, NG at a time
      constexpr int MINE = 4 / S::TG, NG = MINE < 2 ? MINE : 2;
#pragma unroll 1
      for (int g0 = tg * MINE; g0 < (tg + 1) * MINE; g0 += NG) {
        if (16 * g0 < rows) {
          float acc[2][2 * NG][4] = {};
          if (!zero_state) {
#pragma unroll
            for (int ks = 0; ks < DK / 16; ++ks) {
              uint32_t a[NP][4];
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                uint32_t w[NP];
                mma::split2<NP>(st[(2 * ks + (y >> 1)) % (2 * S::N2)][2 * (y & 1)],
                                st[(2 * ks + (y >> 1)) % (2 * S::N2)][2 * (y & 1) + 1], w);
#pragma unroll
                for (int s = 0; s < NP; ++s) a[s][y] = w[s];
              }
#pragma unroll
              for (int n2 = 0; n2 < NG; ++n2) {
                uint32_t bf[NP][4];
#pragma unroll
                for (int s = 0; s < NP; ++s)
                  mma::ldsm4(bf[s], Qs + s * (C * DK * 2) +
                                        mma::tile_off<DK>(16 * (g0 + n2) + (m >> 1) * 8 + r8, 2 * ks + (m & 1)));
#pragma unroll
                for (int sa = NP - 1; sa >= 0; --sa)
#pragma unroll
                  for (int sb = NP - 1 - sa; sb >= 0; --sb) {
                    mma::mma16816(acc[sa + sb > 0][2 * n2], a[sa], bf[sb][0], bf[sb][1]);
                    mma::mma16816(acc[sa + sb > 0][2 * n2 + 1], a[sa], bf[sb][2], bf[sb][3]);
                  }
              }
            }
#pragma unroll
            for (int n = 0; n < 2 * NG; ++n)
#pragma unroll
              for (int y = 0; y < 2; ++y) {
                const float f = P.b * pw[16 * g0 + 8 * n + 2 * t + y + 1 - P.e];
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                  acc[w][n][y] *= f;
                  acc[w][n][y + 2] *= f;
                }
              }
          }
          if (!odd) {
#pragma unroll
            for (int kb16 = 0; kb16 < 4; ++kb16) {
              if (kb16 < g0 + NG) {
                uint32_t a[NP][4];
#pragma unroll
                for (int s = 0; s < NP; ++s)
                  mma::ldsm4t(a[s], Vs + s * (C * DV * 2) +
                                        mma::tile_off<DV>(16 * kb16 + (m >> 1) * 8 + r8, row / 8 + (m & 1)));
#pragma unroll
                for (int n2 = 0; n2 < NG; ++n2) {
                  if (kb16 <= g0 + n2) {  // scores beyond are 0
                    uint32_t bf[NP][4];
#pragma unroll
                    for (int s = 0; s < NP; ++s)
                      mma::ldsm4(bf[s], Pa + s * (C * C * 2) +
                                            mma::tile_off<C>(16 * (g0 + n2) + (m >> 1) * 8 + r8, 2 * kb16 + (m & 1)));
#pragma unroll
                    for (int sa = NP - 1; sa >= 0; --sa)
#pragma unroll
                      for (int sb = NP - 1 - sa; sb >= 0; --sb) {
                        mma::mma16816(acc[sa + sb > 0][2 * n2], a[sa], bf[sb][0], bf[sb][1]);
                        mma::mma16816(acc[sa + sb > 0][2 * n2 + 1], a[sa], bf[sb][2], bf[sb][3]);
                      }
                  }
                }
              }
            }
          } else {
            float by_term[2 * NG][4];  // (not acc itself: what a call gets by address lies in memory throughout)
            slow_pv<DV, 2 * NG>(by_term, Ps, Vc, 16 * g0, row);
#pragma unroll
            for (int n = 0; n < 2 * NG; ++n)
#pragma unroll
              for (int x = 0; x < 4; ++x) acc[0][n][x] += by_term[n][x];
          }
          // o^T -> o: element (token 2t, 2t + 1; value row g, g + 8)
#pragma unroll
          for (int n = 0; n < 2 * NG; ++n)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int i = 16 * g0 + 8 * n + 2 * t + (x & 1), vr = row + g + 8 * (x >> 1);
              if (i < rows && vr < P.vd) {
                const int64_t tok = bi * A.T + first + step * (c * C + i);
                static_cast<float*>(P.o)[(tok * A.H + h) * P.vd + vr] = acc[0][n][x] + acc[1][n][x];
              }
            }
        }
      }
    }

    // the state behind this block
    if (owner && (STATE_ONLY || c + 1 < blocks || (P.seg == nullptr && P.fin != nullptr))) {
      const float keep = pw[rows];
#pragma unroll
      for (int p2 = 0; p2 < 2; ++p2) {  // tokens 0..31 and 32..63
        if (32 * p2 < rows) {
          uint32_t a[2][NP][4];
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
              uint32_t w[NP];
              mma::split2<NP>(va[y][0] * f0, va[y][1] * f1, w);
#pragma unroll
              for (int s = 0; s < NP; ++s) a[q2][s][y] = w[s];
            }
          }
#pragma unroll
          for (int n2 = 0; n2 < S::N2; ++n2) {
            float add[2][2][4] = {};  // first parts' products; the others'
#pragma unroll
            for (int q2 = 0; q2 < 2; ++q2) {
              uint32_t bf[NP][4];
#pragma unroll
              for (int s = 0; s < NP; ++s)
                mma::ldsm4t(bf[s], Ks + s * (C * DK * 2) +
                                       mma::tile_off<DK>(32 * p2 + 16 * q2 + (m & 1) * 8 + r8, col0 / 8 + 2 * n2 + (m >> 1)));
#pragma unroll
              for (int sb = 0; sb < NP; ++sb)
#pragma unroll
                for (int sa = NP - 1 - sb; sa >= 0; --sa) {
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
  else if (P.seg == nullptr && P.fin != nullptr && tg == 0)  // every token group has the same state
    dst = P.fin + sbase;
  if (dst != nullptr && owner) {
#pragma unroll
    for (int n = 0; n < 2 * S::N2; ++n)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int kr = col0 + 8 * n + 2 * t + (x & 1), vr = row + g + 8 * (x >> 1);
        if (kr < P.kd && vr < P.vd) dst[static_cast<int64_t>(kr) * P.vd + vr] = st[n][x];
      }
  }
}

}  // namespace da
}  // namespace ttc
