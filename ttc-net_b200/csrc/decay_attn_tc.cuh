// The recurrence of decay_attn.cuh for bf16 on the 5th-generation tensor cores: one persistent-state CTA for
// each segment of a (sequence, head), blocks of 64 tokens, five warpgroups with roles of their own.
//
// Products of a block (M = 128 TMEM lanes; dv or 64 tokens of them used, rows are independent):
//   Sc [i x j]   = q k^T                A = q, B = k                  (shared memory, K-major)
//   U  [dv x dk] = (f v)^T k            A = f v in bf16 parts, B = k  (shared memory, MN-major)
//   O1 [dv x i]  = bf16(S)^T q^T        A = S^T in TMEM, B = q        (K-major)
//   O2 [dv x i]  = v^T P^T              A = v (MN-major), B = P       (K-major)
// One shared-memory image of a tile serves as K-major and as MN-major operand: halves of 64 columns, rows of
// 128 bytes, 16-byte pieces xor-ed with the row (the 128-byte swizzle).
//
// Roles:
//   warps 0-3    the state: row dv of S^T in DK fp32 registers of its thread, S = gamma^rows S + U
//                with an ordinary fma (U is summed from zero in TMEM), and S in bf16 to TMEM
//   warps 4-7    o = f_i O1 + O2, rounded and staged through the block's v tile to 16-byte stores
//   warps 8, 9   P = scores times decays, masked, in bf16 to shared memory
//   warp 10      issues every tcgen05.mma
//   warps 12-15  f v in two or three bf16 parts; notes blocks whose v holds Inf or NaN
//   warps 16-18  16-byte asynchronous copies of every third block each (three stages)
// Every wait is bounded (about two seconds); one that runs out makes all roles leave and sets
// TTC_STATUS_MMA_TIMEOUT in the status word.
#pragma once

#include "decay_attn.cuh"
#include "tc_primitives.cuh"
#include "ttc_b200.h"

namespace ttc {
namespace da {

constexpr int kTcThreads = 640, kTcStages = 3;

template <int DK, int DV>
struct TcShape {
  static constexpr int KB = C * DK * 2, VB = C * DV * 2;
  static constexpr int STAGE = 2 * KB + VB;  // q, k, v
  static constexpr int PB = C * C * 2;
  static constexpr int PARTS = kTcStages * STAGE;  // f v, part by part
  __host__ __device__ static constexpr int p_off(int parts) { return PARTS + parts * VB; }
  __host__ __device__ static constexpr int tail_off(int parts) { return p_off(parts) + 2 * PB; }
  static constexpr int smem(int parts) { return 1024 + tail_off(parts) + 1024; }
  // TMEM columns
  static constexpr int U = 0, S = 128, SC = 192, O = 256;  // O: two buffers of (O1 64, O2 64)
};

struct TcBars {
  uint64_t full[kTcStages], empty[kTcStages], sc_full, sc_empty, p_full[2], p_empty[2], vs_full, vs_empty, u_full,
      u_empty, s_full, s_empty, o_full[2], o_empty[2];
};

// Instruction descriptor: D fp32, A and B bf16, M = 128; *_mn: that operand is MN-major.
__host__ __device__ constexpr uint32_t idesc_bf16(int n, bool a_mn, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) |
         (static_cast<uint32_t>(n >> 3) << 17) | (8u << 24);
}
// Shared-memory descriptor, 128-byte swizzle: 8-row groups 1024 bytes apart, 64-column halves 8192.
__device__ __forceinline__ uint64_t desc128(uint32_t addr) {
  return static_cast<uint64_t>((addr >> 4) & 0x3fffu) | (static_cast<uint64_t>(8192 >> 4) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) | (static_cast<uint64_t>(2) << 61);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, q;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, q;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(tc::smem_u32(bar)) : "memory");
}

// Phase `parity` of `bar`, for a whole warp: false for all lanes once the time is up or another role has given up.
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, volatile int* gone) {
  const uint32_t addr = tc::smem_u32(bar);
  uint64_t t0 = 0;
  for (;;) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 10000;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(addr), "r"(parity)
        : "memory");
    if (__all_sync(0xffffffffu, done)) return true;
    const uint64_t t = tc::global_ns();
    if (t0 == 0) t0 = t;
    if (t - t0 > 2000000000ull) *gone = 1;
    if (__any_sync(0xffffffffu, *gone != 0)) return false;
  }
}

template <int N>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

__device__ __forceinline__ uint32_t swz(int r, int c) { return static_cast<uint32_t>(r * 128 + ((c ^ (r & 7)) << 4)); }
__device__ __forceinline__ float bf_at(const char* tile, int r, int col) {
  return __bfloat162float(
      *reinterpret_cast<const __nv_bfloat16*>(tile + (col >> 6) * 8192 + swz(r, (col & 63) >> 3) + (col & 7) * 2));
}

template <int DK, int DV, bool STATE_ONLY>
__global__ void __launch_bounds__(kTcThreads, 1) decay_attn_tc_kernel(const __grid_constant__ Args A, int* status) {
  using S = TcShape<DK, DV>;
  extern __shared__ char smem_raw[];
  __shared__ TcBars bars;
  __shared__ uint32_t tmem_base;
  __shared__ int gone_s, bad_s[kTcStages];
  __shared__ float pw[72];
  char* const smem = smem_raw + ((1024 - (tc::smem_u32(smem_raw) & 1023)) & 1023);
  const Pass& P = A.pass[blockIdx.z];
  const int h = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  if (!STATE_ONLY && A.cu != nullptr && static_cast<int>(blockIdx.x) == A.items) {
    zero_rows_behind<true>(A, P, h, tid, kTcThreads);
    return;
  }
  const Item it = find_item(A, blockIdx.x);
  if (it.seq < 0) return;
  const int64_t s0 = static_cast<int64_t>(it.seg) * A.seg_len;
  const int64_t left = it.len - s0;
  const int seg_rows = static_cast<int>(left < A.seg_len ? (left > 0 ? left : 0) : A.seg_len);
  const int blocks = (seg_rows + C - 1) / C;
  if (STATE_ONLY && s0 + seg_rows >= it.len && P.fin == nullptr) return;
  const bool keep_last = STATE_ONLY || (P.seg == nullptr && P.fin != nullptr);  // the state behind the last block
  const int parts = A.parts;

  volatile int* const gone = &gone_s;
  if (tid == 0) {
    for (int i = 0; i < kTcStages; ++i) {
      tc::mbar_init(&bars.full[i], 1);
      tc::mbar_init(&bars.empty[i], STATE_ONLY ? 4 : 8);
      bad_s[i] = 0;
    }
    tc::mbar_init(&bars.sc_full, 1);
    tc::mbar_init(&bars.sc_empty, 2);
    tc::mbar_init(&bars.vs_full, 4);
    tc::mbar_init(&bars.vs_empty, 1);
    tc::mbar_init(&bars.u_full, 1);
    tc::mbar_init(&bars.u_empty, 4);
    tc::mbar_init(&bars.s_full, 4);
    tc::mbar_init(&bars.s_empty, 1);
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&bars.p_full[i], 2);
      tc::mbar_init(&bars.p_empty[i], 4);
      tc::mbar_init(&bars.o_full[i], 1);
      tc::mbar_init(&bars.o_empty[i], 4);
    }
    gone_s = 0;
    tc::mbar_init_fence();
  }
  if (tid >= 64 && tid <= 64 + C) pw[tid - 64] = decay_pow(A.log_gamma[h], tid - 64);
  if (warp == 11) tc::tmem_alloc(&tmem_base, 512);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tm = tmem_base;
  const int64_t sbase = (static_cast<int64_t>(it.seq) * A.H + h) * P.kd * P.vd;
  const int64_t gbase = ((it.index + it.seg) * A.H + h) * P.kd * P.vd;

  if (warp < 4) {  // ---------------------------------------------------------------- the state
    regs_inc<192>();
    const uint32_t my = tm + (static_cast<uint32_t>(warp * 32) << 16);
    const int vr = warp * 32 + lane;
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
    float st[DK];
#pragma unroll
    for (int k = 0; k < DK; ++k) st[k] = src != nullptr && k < P.kd && vr < P.vd ? src[k * sk + vr * sv] : 0.f;
    for (int c = 0; c < blocks; ++c) {
      const int rows = min(C, seg_rows - c * C);
      if (!STATE_ONLY) {
        if (c > 0 && !wait_bar(&bars.s_empty, (c - 1) & 1, gone)) break;
        tc::fence_after_sync();
#pragma unroll
        for (int x = 0; x < DK / 64; ++x) {
          float w[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) w[i] = __uint_as_float(mma::pack2(st[64 * x + 2 * i], st[64 * x + 2 * i + 1]));
          tc::tmem_st<32>(my + S::S + 32 * x, w);
        }
        tc::tmem_wait_st();
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.s_full);
      }
      if (c + 1 < blocks || keep_last) {
        if (!wait_bar(&bars.u_full, c & 1, gone)) break;
        tc::fence_after_sync();
        const float keep = pw[rows];
#pragma unroll
        for (int x = 0; x < DK / 32; ++x) {
          float u[32];
          tc::tmem_ld<32>(my + S::U + 32 * x, u);
#pragma unroll
          for (int i = 0; i < 32; ++i) st[32 * x + i] = fmaf(keep, st[32 * x + i], u[i]);
        }
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bars.u_empty);
          mbar_arrive(&bars.empty[c % kTcStages]);
        }
      }
    }
    float* dst = nullptr;
    if (STATE_ONLY)
      dst = P.seg + gbase;
    else if (keep_last)
      dst = P.fin + sbase;
    if (dst != nullptr && vr < P.vd) {
#pragma unroll
      for (int k = 0; k < DK; ++k)
        if (k < P.kd) dst[static_cast<int64_t>(k) * P.vd + vr] = st[k];
    }
  } else if (warp < 8) {  // ------------------------------------------------------------ the outputs
    if (!STATE_ONLY) {
      const int w4 = warp - 4, vr = w4 * 32 + lane, t4 = tid - 128;
      const uint32_t my = tm + (static_cast<uint32_t>(w4 * 32) << 16);
      const int bi = A.cu == nullptr ? it.seq : 0;
      const int64_t step = P.reverse ? -1 : 1;
      const int64_t tok0 = bi * A.T + it.row0 + (P.reverse ? it.len - 1 - s0 : s0);
      const bool live = w4 * 32 < P.vd;
      for (int c = 0; c < blocks; ++c) {
        const int rows = min(C, seg_rows - c * C), s = c % kTcStages, b = c & 1;
        if (!wait_bar(&bars.o_full[b], (c >> 1) & 1, gone)) break;
        tc::fence_after_sync();
        char* const vt = smem + s * S::STAGE + 2 * S::KB;
        const bool bad = *static_cast<volatile int*>(&bad_s[s]) == c + 1;
        uint32_t out[2][16];
        float* const of = static_cast<float*>(P.o);
        const char* const pt = smem + S::p_off(parts) + b * S::PB;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float o1[32], o2[32];
          tc::tmem_ld<32>(my + S::O + 128 * b + 32 * x, o1);
          tc::tmem_ld<32>(my + S::O + 128 * b + 64 + 32 * x, o2);
          if (bad) {  // 0 * NaN: term by term over j <= i
#pragma unroll 1
            for (int i = 0; i < 32; ++i) {
              float a = 0.f;
              for (int j = 0; j <= 32 * x + i; ++j)
                if (vr < P.vd) a = fmaf(bf_at(pt, 32 * x + i, j), bf_at(vt, j, vr), a);
              // registers are indexed by constants only
#pragma unroll
              for (int q = 0; q < 32; ++q)
                if (q == i) o2[q] = a;
            }
          }
#pragma unroll
          for (int i = 0; i < 32; ++i) o1[i] = fmaf(P.b * pw[32 * x + i + 1 - P.e], o1[i], o2[i]);
          if (P.o_f32) {
            if (vr < P.vd) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (32 * x + i < rows)
                  of[((tok0 + step * (c * C + 32 * x + i)) * A.H + h) * P.vd + vr] = o1[i];
            }
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) out[x][i] = mma::pack2(o1[2 * i], o1[2 * i + 1]);
          }
        }
        tc::fence_before_sync();
        if (bad) tc::named_sync(1, 128);  // all of v is read before it is overwritten
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bars.o_empty[b]);
          mbar_arrive(&bars.p_empty[b]);
        }
        if (!P.o_f32) {
          // rows of DV values; the last readers of the v tile are done (this block's O2)
          if (live) {
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                char* p = vt + (32 * x + 2 * i) * (DV * 2) + vr * 2;
                *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(out[x][i]);
                *reinterpret_cast<uint16_t*>(p + DV * 2) = static_cast<uint16_t>(out[x][i] >> 16);
              }
          }
          tc::named_sync(1, 128);
          __nv_bfloat16* const ob = static_cast<__nv_bfloat16*>(P.o);
          for (int x = t4; x < C * (DV / 8); x += 128) {
            const int i = x / (DV / 8), p8 = x % (DV / 8);
            if (i < rows && p8 * 8 < P.vd)
              *reinterpret_cast<uint4*>(ob + ((tok0 + step * (c * C + i)) * A.H + h) * P.vd + p8 * 8) =
                  *reinterpret_cast<const uint4*>(vt + i * (DV * 2) + p8 * 16);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.empty[s]);
      }
    }
  } else if (warp < 12) {
    regs_dec<64>();
    if (warp < 10) {  // ---------------------------------------------------------------- the scores
      if (!STATE_ONLY) {
        const int i = (warp - 8) * 32 + lane;
        const uint32_t my = tm + (static_cast<uint32_t>((warp - 8) * 32) << 16) + S::SC;
        for (int c = 0; c < blocks; ++c) {
          const int b = c & 1;
          if (c > 1 && !wait_bar(&bars.p_empty[b], ((c >> 1) - 1) & 1, gone)) break;
          if (!wait_bar(&bars.sc_full, c & 1, gone)) break;
          tc::fence_after_sync();
          char* const pt = smem + S::p_off(parts) + b * S::PB;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float v[32];
            tc::tmem_ld<32>(my + 32 * x, v);
            if (x == 1) {
              tc::fence_before_sync();
              __syncwarp();
              if (lane == 0) mbar_arrive(&bars.sc_empty);
            }
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              uint32_t w[4];
#pragma unroll
              for (int z = 0; z < 4; ++z) {
                const int j = 32 * x + 8 * y + 2 * z, e = 8 * y + 2 * z;
                const float v0 = j <= i ? v[e] * (P.a * pw[max(i - j, 0)]) : 0.f;
                const float v1 = j + 1 <= i ? v[e + 1] * (P.a * pw[max(i - j - 1, 0)]) : 0.f;
                w[z] = mma::pack2(v0, v1);
              }
              *reinterpret_cast<uint4*>(pt + swz(i, 4 * x + y)) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
          tc::fence_smem_to_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars.p_full[b]);
        }
      }
    } else if (warp == 10) {  // ------------------------------------------------------------- the MMAs
      const uint32_t base = tc::smem_u32(smem);
      const int kd16 = (P.kd + 15) / 16;
      constexpr uint32_t d_sc = idesc_bf16(64, false, false), d_u = idesc_bf16(DK, true, true),
                         d_o2 = idesc_bf16(64, true, false);
      auto scores = [&](int c) {
        const uint32_t q = base + (c % kTcStages) * S::STAGE, k = q + S::KB;
        if (!wait_bar(&bars.full[c % kTcStages], (c / kTcStages) & 1, gone)) return false;
        if (c > 0 && !wait_bar(&bars.sc_empty, (c - 1) & 1, gone)) return false;
        tc::fence_after_sync();
        if (lane == 0) {
          for (int x = 0; x < kd16; ++x) {
            const uint32_t off = (x >> 2) * 8192 + (x & 3) * 32;
            mma_ss(tm + S::SC, desc128(q + off), desc128(k + off), d_sc, x > 0);
          }
          tc::mma_commit(&bars.sc_full);
        }
        __syncwarp();
        return true;
      };
      bool ok = STATE_ONLY || blocks == 0 || scores(0);
      for (int c = 0; ok && c < blocks; ++c) {
        const int s = c % kTcStages, b = c & 1;
        const uint32_t q = base + s * S::STAGE, k = q + S::KB, v = k + S::KB;
        if (!(ok = wait_bar(&bars.vs_full, c & 1, gone))) break;
        if (c + 1 < blocks || keep_last) {
          if (c > 0 && !(ok = wait_bar(&bars.u_empty, (c - 1) & 1, gone))) break;
          tc::fence_after_sync();
          if (lane == 0) {
            for (int p = parts - 1; p >= 0; --p)
              for (int x = 0; x < C / 16; ++x)
                mma_ss(tm + S::U, desc128(base + S::PARTS + p * S::VB + x * 2048), desc128(k + x * 2048), d_u,
                       p < parts - 1 || x > 0);
            tc::mma_commit(&bars.vs_empty);
            tc::mma_commit(&bars.u_full);
          }
          __syncwarp();
        }
        if (STATE_ONLY) continue;
        if (!(ok = wait_bar(&bars.s_full, c & 1, gone))) break;
        if (c > 1 && !(ok = wait_bar(&bars.o_empty[b], ((c >> 1) - 1) & 1, gone))) break;
        tc::fence_after_sync();
        if (lane == 0) {
          for (int x = 0; x < kd16; ++x)
            mma_ts(tm + S::O + 128 * b, tm + S::S + x * 8, desc128(q + (x >> 2) * 8192 + (x & 3) * 32), d_sc, x > 0);
          tc::mma_commit(&bars.s_empty);
        }
        __syncwarp();
        if (c + 1 < blocks && !(ok = scores(c + 1))) break;
        if (!(ok = wait_bar(&bars.p_full[b], (c >> 1) & 1, gone))) break;
        tc::fence_after_sync();
        if (lane == 0) {
          const uint32_t p = base + S::p_off(parts) + b * S::PB;
          for (int x = 0; x < C / 16; ++x)
            mma_ss(tm + S::O + 128 * b + 64, desc128(v + x * 2048), desc128(p + x * 32), d_o2, x > 0);
          tc::mma_commit(&bars.o_full[b]);
        }
        __syncwarp();
      }
    }
  } else if (warp < 16) {  // ----------------------------------------------------- the decayed values
    regs_dec<64>();
    const int t4 = tid - 384;
    for (int c = 0; c < blocks; ++c) {
      const int rows = min(C, seg_rows - c * C), s = c % kTcStages;
      if (!wait_bar(&bars.full[s], (c / kTcStages) & 1, gone)) break;
      const bool update = c + 1 < blocks || keep_last;
      if (c > 0 && !wait_bar(&bars.vs_empty, (c - 1) & 1, gone)) break;
      const char* const vt = smem + s * S::STAGE + 2 * S::KB;
      float chk = 0.f;
#pragma unroll 2
      for (int x = t4; x < C * DV / 8; x += 128) {
        const int half = x / 512, r = (x >> 3) & 63;
        const uint32_t off = half * 8192 + swz(r, x & 7);
        const uint4 w = *reinterpret_cast<const uint4*>(vt + off);
        const float f = r < rows ? P.u * pw[max(rows - 1 - r + P.e, 0)] : 0.f;
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
        uint32_t o[4][3];
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const float a = mma::lo_f(u[y]), d = mma::hi_f(u[y]);
          chk = fmaf(a, 0.f, fmaf(d, 0.f, chk));
          mma::split2<3>(a * f, d * f, o[y]);
        }
        if (update) {
          for (int p = 0; p < 3; ++p)
            if (p < parts)
              *reinterpret_cast<uint4*>(smem + S::PARTS + p * S::VB + off) =
                  make_uint4(o[0][p], o[1][p], o[2][p], o[3][p]);
        }
      }
      if (chk != 0.f) *static_cast<volatile int*>(&bad_s[s]) = c + 1;  // NaN too
      tc::fence_smem_to_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.vs_full);
    }
  } else {
    regs_dec<64>();
    if (warp < 16 + kTcStages) {  // ------------------------------------------------------- the copies
      const int s = warp - 16;
      const int bi = A.cu == nullptr ? it.seq : 0;
      const char* qb = static_cast<const char*>(P.q) + (bi * P.qs[0] + (h / P.qg) * P.qs[2]) * 2;
      const char* kb = static_cast<const char*>(P.k) + (bi * P.ks[0] + (h / P.kg) * P.ks[2]) * 2;
      const char* vb = static_cast<const char*>(P.v) + (bi * P.vs[0] + (h / P.vg) * P.vs[2]) * 2;
      const int64_t step = P.reverse ? -1 : 1;
      const int64_t first = it.row0 + (P.reverse ? it.len - 1 - s0 : s0);
      const uint32_t base = tc::smem_u32(smem) + s * S::STAGE;
      const int piece = lane & 7, r4 = lane >> 3;
      // rows r4, r4 + 4, ... of a tile: 8 lanes copy a row's 128 bytes of one half
      auto tile = [&](uint32_t dst, const char* src, int64_t row_stride, int halves, int d, int64_t f, int rows) {
        for (int hf = 0; hf < halves; ++hf) {
          const bool col = hf * 64 + piece * 8 < d;
          const char* p = src + ((f + step * r4) * row_stride + hf * 64 + piece * 8) * 2;
          const int64_t next = step * row_stride * 8;
#pragma unroll 4
          for (int r = r4; r < C; r += 4) {
            const bool on = col && r < rows;
            mma::cp16(dst + hf * 8192 + swz(r, piece), on ? p : src, on ? 16 : 0);
            p += next;
          }
        }
      };
      for (int c = s; c < blocks; c += kTcStages) {
        const int rows = min(C, seg_rows - c * C);
        if (c >= kTcStages && !wait_bar(&bars.empty[s], ((c / kTcStages) - 1) & 1, gone)) break;
        const int64_t f = first + step * c * C;
        if (!STATE_ONLY) tile(base, qb, P.qs[1], DK / 64, P.kd, f, rows);
        tile(base + S::KB, kb, P.ks[1], DK / 64, P.kd, f, rows);
        tile(base + 2 * S::KB, vb, P.vs[1], DV / 64, P.vd, f, rows);
        mma::cp_commit();
        mma::cp_wait<0>();
        tc::fence_smem_to_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.full[s]);
      }
      mma::cp_wait<0>();
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  if (warp == 11) tc::tmem_dealloc(tm, 512);
  if (tid == 0 && gone_s != 0 && status != nullptr) atomicOr_system(status, TTC_STATUS_MMA_TIMEOUT);
}

}  // namespace da
}  // namespace ttc
