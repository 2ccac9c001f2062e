// The recurrence of decay_attn.cuh for bf16 on the 5th-generation tensor cores: one persistent-state CTA for
// each segment of a (sequence, head), blocks of 64 tokens, five warpgroups with roles of their own.
//
// Products of a block (M = 128 TMEM lanes, dv of them used, rows are independent; M = 64 for the scores):
//   Sc [i x j]   = q k^T                A = q, B = k                  (shared memory, K-major)
//   U  [dv x dk] = (f v)^T k            A = (f v)^T in bf16 parts in TMEM, B = k (shared memory, MN-major)
//   O1 [dv x i]  = bf16(S)^T q^T        A = S^T in TMEM, B = q        (K-major)
//   O2 [dv x i]  = v^T P^T              A = v (MN-major), B = P       (K-major)
// One shared-memory image of a tile serves as K-major and as MN-major operand: halves of 64 columns, rows of
// 128 bytes, 16-byte pieces xor-ed with the row (the 128-byte swizzle).
//
// Roles:
//   warps 0-3    the state: row dv of S^T in DK fp32 registers of its thread, S = gamma^rows S + U
//                with an ordinary fma (U is summed from zero in TMEM), and S in bf16 to TMEM
//   warps 4-7    o = f_i O1 + O2, rounded, transposed through shared memory to 16-byte stores
//   warps 8-15   (f v)^T in two or three bf16 parts to TMEM; note blocks whose v holds Inf or NaN
//   warps 8-11   also P = scores times decays, masked, in bf16 to shared memory
//   warp 16      copies by TMA, four to six blocks ahead; zeros in what a sequence's partial last block
//                holds of others
//   warps 18, 19 issue the tcgen05.mma's: scores and outputs, and U (one thread for all was the longest chain)
// What bounds it at 128 x 128 is shared memory: 208 KB of reads and writes a block, 1 600 cycles of its 128 bytes a
// cycle (272 KB with the parts of f v in shared memory too), then the chain load - parts - U and scores - O2 a
// stage is held for.
// Roundings below fp32: the scores times decays and the copy of the state that q multiplies go to bf16 once each, as the
// outputs do behind them (2.3e-3 from the exact outputs in all, 1.7e-3 of it the outputs' own rounding); the state itself
// stays in fp32, and the decayed values that update it come in two bf16 parts (16 bits, below what an output shows), or
// three (24 bits) where the last state is asked for (1e-7 to 2e-7 of it).
// Measured at full clock: 8 x 4096 tokens, 32 heads of 128: 234 us (4.6 TB/s), 258 with last states, 307 in a long run,
// where the board reaches its power limit; 4 x 4096, 37 heads (one CTA on each SM) 122 us, 5.1 TB/s; 37 heads of 64:
// 106 us.  A CTA of one block takes 6 us, of which starting and ending are four: packed prompts of a few blocks each
// are bound by that (a form with CTAs that go on with further pieces made every block 7 % slower and was no faster on
// them).
// Rows of a block lie in token order; in a backward pass the later row is the earlier place.
// Every wait is bounded (wait_bar); one that runs out makes all roles leave and sets
// TTC_STATUS_MMA_TIMEOUT in the status word.
#pragma once

#include <cuda.h>

#include <type_traits>

#include "decay_attn.cuh"
#include "tc_primitives.cuh"
#include "ttc_b200.h"

namespace ttc {
namespace da {

constexpr int kTcThreads = 640;

template <int DK, int DV>
struct TcShape {
  static constexpr int KB = C * DK * 2, VB = C * DV * 2;
  static constexpr int STAGE = 2 * KB + VB;  // q, k, v
  static constexpr int STAGES = DK + DV <= 128 ? 6 : 4;
  static constexpr int PB = C * C * 2;
  static constexpr int P_OFF = STAGES * STAGE;  // two blocks' P
  static constexpr int O_OFF = P_OFF + 2 * PB;  // a block's outputs on their way
  static constexpr int SMEM = 1024 + O_OFF + VB;
  // TMEM columns: U, bf16(S), scores, O1 and O2, the parts of f v
  static constexpr int U = 0, S = 128, SC = 192, O = 256, F = 384;
};

template <int STAGES>
struct TcBars {
  uint64_t full[STAGES], empty[STAGES], noted[STAGES], part, sc_full, sc_empty, p_full[2], p_empty[2], vs_full[2], vs_empty[2], u_full, u_empty,
      s_full, s_empty, o_full, o_empty;
};

// Tensor maps [batch, head, token, dim], boxes of 64 tokens x 64 dims, 128-byte swizzle: a pass reads q, k, v
// through maps number m[pass][0 .. 2] and writes o, where that is bf16, through out[pass].
struct TcMaps {
  CUtensorMap map[4], out[3];
  int m[3][3];
};

__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, int x, int row, int head, int batch,
                                        uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(dst),
      "l"(map), "r"(x), "r"(row), "r"(head), "r"(batch), "r"(tc::smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void mbar_expect(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(tc::smem_u32(bar)), "r"(bytes) : "memory");
}

// Instruction descriptor: D fp32, A and B bf16; *_mn: that operand is MN-major.
__host__ __device__ constexpr uint32_t idesc_bf16(int m, int n, bool a_mn, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) |
         (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
// Shared-memory descriptor, 128-byte swizzle, 8-row groups 1024 bytes apart, 64-column halves 8192: the
// upper word is a constant, the lower one moves by bytes / 16.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr) { return (addr >> 4) | ((8192u >> 4) << 16); }
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 q, %4, 0;\n\t"
      "mov.b64 x, {%1, %5};\n\tmov.b64 y, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, q;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "n"(kDescHi)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t.reg .b64 y;\n\tsetp.ne.b32 q, %4, 0;\n\tmov.b64 y, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, q;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "n"(kDescHi)
      : "memory");
}
// 16 lanes x 64 columns in the layout of mma accumulators: v[4 n + x] is lane g + 8 (x >> 1), column
// 8 n + 2 t + (x & 1) of thread (g, t) = (lane / 4, lane % 4).  No wait.
__device__ __forceinline__ void tmem_ld_frag(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"
      "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
        "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),
        "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_wait_ld(float (&a)[32], float (&b)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
  // the loaded registers are not to be read before the wait
#pragma unroll
  for (int i = 0; i < 32; ++i) asm volatile("" : "+f"(a[i]), "+f"(b[i]));
}
// The same for 16 columns.
__device__ __forceinline__ void tmem_ld_frag(uint32_t taddr, float (&v)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_wait_ld(float (&a)[8]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 8; ++i) asm volatile("" : "+f"(a[i]));
}
// Four 8x8 matrices of 16-bit values.
__device__ __forceinline__ void stsm4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c),
               "r"(d)
               : "memory");
}
// The same, each stored transposed.
__device__ __forceinline__ void stsm4t(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b),
               "r"(c), "r"(d)
               : "memory");
}
// (a, b) = (x, y) (a, b) + (c, d), rounded as two fmas.
__device__ __forceinline__ void fma2(float& a, float& b, float x, float y, float c, float d) {
  asm("{\n\t.reg .b64 p, q, r;\n\tmov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %3};\n\tmov.b64 r, {%4, %5};\n\t"
      "fma.rn.f32x2 p, p, q, r;\n\tmov.b64 {%0, %1}, p;\n\t}"
      : "+f"(a), "+f"(b)
      : "f"(x), "f"(y), "f"(c), "f"(d));
}
__device__ __forceinline__ void tma_out(const CUtensorMap* map, uint32_t src, int x, int row, int head, int batch) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(map), "r"(src),
               "r"(x), "r"(row), "r"(head), "r"(batch)
               : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
// PARTS bf16 parts of (f, h) times the two bf16 values in u (no care for Inf: such blocks are noted anyway).
template <int PARTS>
__device__ __forceinline__ void decayed(uint32_t u, float f, float h, uint32_t (&o)[PARTS]) {
  float x, y;
  asm("{\n\t.reg .b64 p, q;\n\tmov.b64 p, {%2, %3};\n\tmov.b64 q, {%4, %5};\n\tmul.rn.f32x2 p, p, q;\n\t"
      "mov.b64 {%0, %1}, p;\n\t}"
      : "=f"(x), "=f"(y)
      : "f"(mma::lo_f(u)), "f"(mma::hi_f(u)), "f"(f), "f"(h));
#pragma unroll
  for (int p = 0; p < PARTS; ++p) {
    o[p] = mma::pack2(x, y);
    if (p + 1 < PARTS)
      asm("{\n\t.reg .b64 p, q;\n\tmov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %3};\n\tsub.rn.f32x2 p, p, q;\n\t"
          "mov.b64 {%0, %1}, p;\n\t}"
          : "+f"(x), "+f"(y)
          : "f"(mma::lo_f(o[p])), "f"(mma::hi_f(o[p])));
  }
}
// 16 lanes x 8 columns from ldmatrix's registers: a, b the lanes 0-7 and 8-15 of columns 0-3, c, d of 4-7.
__device__ __forceinline__ void tmem_st_frag(uint32_t taddr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x2.b32 [%0], {%1,%2,%3,%4};" ::"r"(taddr), "r"(a), "r"(b), "r"(c), "r"(d)
               : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(tc::smem_u32(bar)) : "memory");
}

__device__ __forceinline__ uint32_t bar_try(uint32_t addr, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 1000;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(addr), "r"(parity)
      : "memory");
  return done;
}
// Phase `parity` of `bar`, for a whole warp: false for all lanes after two million polls (each sleeps up to a
// microsecond) or once another role has given up.
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, volatile int* gone) {
  const uint32_t addr = tc::smem_u32(bar);
#pragma unroll 1
  for (int n = 0; n < 2000000; ++n) {
    if (__all_sync(0xffffffffu, bar_try(addr, parity))) return true;
    if (__any_sync(0xffffffffu, *gone != 0)) return false;
  }
  *gone = 1;
  return false;
}

// For one thread alone.
__device__ __forceinline__ bool wait_one(uint64_t* bar, uint32_t parity, volatile int* gone) {
  const uint32_t addr = tc::smem_u32(bar);
#pragma unroll 1
  for (int n = 0; n < 2000000; ++n) {
    if (bar_try(addr, parity)) return true;
    if (*gone != 0) return false;
  }
  *gone = 1;
  return false;
}
// Named barrier that tells every thread whether all of them had `ok`.
__device__ __forceinline__ bool sync_all(int id, int count, bool ok) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.and.pred q, %2, %3, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"(static_cast<uint32_t>(ok)), "r"(id), "r"(count)
      : "memory");
  return all != 0;
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

__device__ __forceinline__ float tmem_ld_one(uint32_t taddr) {
  uint32_t r;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n\ttcgen05.wait::ld.sync.aligned;" : "=r"(r) : "r"(taddr) : "memory");
  return __uint_as_float(r);
}

// The outputs of a warp's 32 value rows where v holds Inf or NaN, whose products with masked zeros are NaN: the
// scores' product term by term over the past tokens only.  Lane l: value row v0 + l.
__device__ __noinline__ void outputs_by_term(const Pass& P, uint32_t o1, const char* pt, const char* vt, const float* pw,
                                             int v0, int lo, int hi, int64_t at, int64_t row) {
  const int vr = v0 + (threadIdx.x & 31);
#pragma unroll 1
  for (int i = 0; i < C; ++i) {
    __syncwarp();
    const float o = tmem_ld_one(o1 + i);
    if (vr < P.vd && i >= lo && i < hi) {
      float a = 0.f;
#pragma unroll 1
      for (int j = P.reverse ? i : 0; j <= (P.reverse ? C - 1 : i); ++j) a = fmaf(bf_at(pt, i, j), bf_at(vt, j, vr), a);
      a = fmaf(P.b * pw[(P.reverse ? C - 1 - i : i) + 1 - P.e], o, a);
      const int64_t e = at + i * row + vr;
      if (P.o_f32)
        static_cast<float*>(P.o)[e] = a;
      else
        static_cast<__nv_bfloat16*>(P.o)[e] = __float2bfloat16_rn(a);
    }
  }
  __syncwarp();
}

template <int DK, int DV, bool STATE_ONLY>
__global__ void __launch_bounds__(kTcThreads, 1) decay_attn_tc_kernel(const __grid_constant__ Args A, const __grid_constant__ TcMaps M, int* status) {
  using S = TcShape<DK, DV>;
  extern __shared__ char smem_raw[];
  constexpr int STAGES = S::STAGES;
  __shared__ TcBars<STAGES> bars;
  __shared__ uint32_t tmem_base;
  __shared__ int gone_s, bad_s[STAGES];
  __shared__ float pw[72];
  char* const smem = smem_raw + ((1024 - (tc::smem_u32(smem_raw) & 1023)) & 1023);
  const Pass& P = A.pass[blockIdx.z];
  const int h = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);

  if (!STATE_ONLY && A.cu != nullptr && static_cast<int>(blockIdx.x) >= A.items) {
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

  const bool rev = P.reverse != 0;
  const int bi = A.cu == nullptr ? it.seq : 0;
  // row of the first block's first row in token order; blocks follow 64 rows up or down
  const int64_t first = rev ? it.row0 + it.len - s0 - C : it.row0 + s0;
  const int64_t down = rev ? -C : C;

  volatile int* const gone = &gone_s;
  if (tid == 0) {
    for (int i = 0; i < STAGES; ++i) {
      tc::mbar_init(&bars.full[i], 1);
      tc::mbar_init(&bars.empty[i], STATE_ONLY ? 4 : 8);
      tc::mbar_init(&bars.noted[i], 8);
      bad_s[i] = 0;
    }
    tc::mbar_init(&bars.part, 1);
    tc::mbar_init(&bars.sc_full, 1);
    tc::mbar_init(&bars.sc_empty, 4);
    tc::mbar_init(&bars.u_full, 1);
    tc::mbar_init(&bars.u_empty, 4);
    tc::mbar_init(&bars.s_full, 4);
    tc::mbar_init(&bars.s_empty, 1);
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&bars.vs_full[i], 4);
      tc::mbar_init(&bars.vs_empty[i], 1);
      tc::mbar_init(&bars.p_full[i], 4);
      tc::mbar_init(&bars.p_empty[i], 4);
    }
    tc::mbar_init(&bars.o_full, 1);
    tc::mbar_init(&bars.o_empty, 4);
    gone_s = 0;
    tc::mbar_init_fence();
  }
  if (tid >= 64 && tid <= 64 + C) pw[tid - 64] = decay_pow(A.log_gamma[h], tid - 64);
  if (warp == 19) tc::tmem_alloc(&tmem_base, 512);
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
    // The initial state comes as a first sum U: 32 values a turn of a rolled loop through TMEM, then the blocks' own
    // update with a factor of 0.  (128 loads in a row took 5 us of a CTA's time, with or without a state, for fetching
    // their code.)
    float st[DK];
#pragma unroll
    for (int k = 0; k < DK; ++k) st[k] = 0.f;
    if (src != nullptr) {
      const float* p = src + vr * sv;
#pragma unroll 1
      for (int k0 = 0; k0 < DK; k0 += 32) {
        float u[32];
#pragma unroll
        for (int i = 0; i < 32; ++i, p += sk) u[i] = k0 + i < P.kd && vr < P.vd ? *p : 0.f;
        tc::tmem_st<32>(my + S::U + k0, u);
      }
      tc::tmem_wait_st();
    }
#pragma unroll 1
    for (int c = -1; c < blocks; ++c) {
      float keep = 0.f;
      if (c >= 0) {
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
        if (c + 1 == blocks && !keep_last) break;
        if (!wait_bar(&bars.u_full, c & 1, gone)) break;
        tc::fence_after_sync();
        keep = pw[min(C, seg_rows - c * C)];
      }
      if (c >= 0 || src != nullptr) {
#pragma unroll
        for (int x = 0; x < DK / 32; ++x) {
          float u[32];
          tc::tmem_ld<32>(my + S::U + 32 * x, u);
#pragma unroll
          for (int i = 0; i < 32; i += 2) fma2(st[32 * x + i], st[32 * x + i + 1], keep, keep, u[i], u[i + 1]);
        }
      }
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&bars.u_empty);
        if (c >= 0) mbar_arrive(&bars.empty[c % STAGES]);
      }
    }
    float* dst = nullptr;
    if (STATE_ONLY)
      dst = P.seg + gbase;
    else if (keep_last)
      dst = P.fin + sbase;
    if (dst != nullptr && vr < P.vd) {
      float* p = dst + vr;
#pragma unroll
      for (int k = 0; k < DK; ++k, p += P.vd)
        if (k < P.kd) *p = st[k];
    }
  } else if (warp < 8) {  // ------------------------------------------------------------ the outputs
    if (!STATE_ONLY) {
      const int w4 = warp - 4, g = lane >> 2, t = lane & 3, m = lane >> 3, r8 = lane & 7, v0 = w4 * 32;
      const uint32_t my = tm + (static_cast<uint32_t>(w4 * 32) << 16) + S::O;
      const uint32_t ot = tc::smem_u32(smem) + S::O_OFF;
      const int64_t row = static_cast<int64_t>(A.H) * P.vd;  // elements between a head's tokens
      int64_t at = (bi * A.T + first) * row + h * static_cast<int64_t>(P.vd);  // the block's first row
      float f[8][2];  // of rows 8 n + 2 t (+ 1)
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int i = 8 * n + 2 * t + x;
          f[n][x] = P.b * pw[(rev ? C - 1 - i : i) + 1 - P.e];
        }
#pragma unroll 1
      for (int c = 0; c < blocks; ++c, at += down * row) {
        const int rows = min(C, seg_rows - c * C), s = c % STAGES, b = c & 1;
        const int lo = rev ? C - rows : 0, hi = lo + rows;  // the block's rows that are in the sequence
        bool ok = wait_bar(&bars.o_full, c & 1, gone);
        // both halves' notes on Inf and NaN; by stage, since those warps may be several blocks ahead
        ok = ok && wait_bar(&bars.noted[s], (c / STAGES) & 1, gone);
        if (tid == 128) bulk_wait_read();  // the staging has left
        // all four warps go on or none
        if (!sync_all(1, 128, ok)) break;
        tc::fence_after_sync();
        const bool bad = *static_cast<volatile int*>(&bad_s[s]) == c + 1;
        if (bad)
          outputs_by_term(P, my, smem + S::P_OFF + b * S::PB, smem + s * S::STAGE + 2 * S::KB, pw, v0, lo,
                          hi, at, row);
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bars.p_empty[b]);
          mbar_arrive(&bars.empty[s]);
        }
        if (!bad) {
#pragma unroll 1
          for (int hl = 0; hl < 2; ++hl) {
            const int vh = v0 + 16 * hl;
            if (vh < P.vd) {
              float o1[32], o2[32];
              tmem_ld_frag(my + (16u << 16) * hl, o1);
              tmem_ld_frag(my + (16u << 16) * hl + 64, o2);
              tmem_wait_ld(o1, o2);
#pragma unroll
              for (int q = 0; q < 32; q += 2) fma2(o1[q], o1[q + 1], f[q >> 2][0], f[q >> 2][1], o2[q], o2[q + 1]);
              if (!P.o_f32) {
#pragma unroll
                for (int n = 0; n < 8; n += 2)
                  stsm4t(ot + (vh >> 6) * 8192 + swz(8 * (n + (m >> 1)) + r8, ((vh & 63) >> 3) + (m & 1)),
                         mma::pack2(o1[4 * n], o1[4 * n + 1]), mma::pack2(o1[4 * n + 2], o1[4 * n + 3]),
                         mma::pack2(o1[4 * n + 4], o1[4 * n + 5]), mma::pack2(o1[4 * n + 6], o1[4 * n + 7]));
              } else {
                float* const of = static_cast<float*>(P.o) + at + vh + g;
                const bool v8 = vh + g + 8 < P.vd;  // widths are multiples of 8: row g is there
#pragma unroll
                for (int q = 0; q < 32; ++q) {
                  const int i = 8 * (q >> 2) + 2 * t + (q & 1);
                  if (i >= lo && i < hi && (!(q & 2) || v8)) of[i * row + 4 * (q & 2)] = o1[q];
                }
              }
            }
          }
        }
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.o_empty);
        if (!P.o_f32 && !bad) {
          tc::fence_smem_to_async();
          tc::named_sync(1, 128);
          if (rows == C) {
            if (tid == 128) {
#pragma unroll
              for (int hf = 0; hf < DV / 64; ++hf)
                if (hf * 64 < P.vd)
                  tma_out(&M.out[blockIdx.z], ot + hf * 8192, hf * 64, static_cast<int>(first + down * c), h, bi);
              bulk_commit();
            }
          } else {  // the rows beyond are not this sequence's
#pragma unroll 1
            for (int x = tid - 128; x < C * DV / 8; x += 128) {
              const int i = x / (DV / 8), p8 = x % (DV / 8);
              if (i >= lo && i < hi && p8 * 8 < P.vd)
                *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(P.o) + at + i * row + p8 * 8) =
                    *reinterpret_cast<const uint4*>(smem + S::O_OFF + (p8 >> 3) * 8192 + swz(i, p8 & 7));
            }
          }
        }
      }
      if (tid == 128) bulk_wait();
    }
  } else if (warp < 16) {  // ------------------------------------------ the decayed values, and the scores
    regs_dec<72>();
    // Warps 8-11 take the block's second 32 tokens' values and then its scores, warps 12-15 the first 32's
    // values: U starts on them one by one, and the tile is held half as long as with one warpgroup.
    // Warp w has value rows (TMEM lanes) 32 w .. 32 w + 31; ldmatrix turns a 16 x 16 corner of v into the layout
    // of a 16-lane TMEM store, two tokens a register: thread (g, t) has tokens 2t, 2t + 1 (+ 8) of rows g (+ 8).
    const int h2 = warp < 12 ? 1 : 0;
    // Scores: warp w has rows 16 w .. 16 w + 15 (M = 64: TMEM lanes 32 w ..), a thread rows g and g + 8, columns
    // 8 n + 2 t + x.  The decay of |i - j| places on the past side (j <= i, or j >= i backwards) is
    // gamma^(whole groups of 8 between them) times a constant of the thread with 1 to 14 places; in the group that
    // holds the diagonal it is `own`, 0 beyond it.  No negative powers, whatever gamma.
    const int w = warp & 3, g = lane >> 2, t = lane & 3, m = lane >> 3, r8 = lane & 7;
    const uint32_t lanes = tm + (static_cast<uint32_t>(w * 32) << 16), my = lanes + S::SC;
    float edge[2], own[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int d = rev ? 2 * t + x - g : g - 2 * t - x;
      edge[x] = pw[8 + d];
      own[x] = d >= 0 ? P.a * pw[max(d, 0)] : 0.f;
    }
    bool see[2] = {rev ? 2 * t >= g : g >= 2 * t, rev ? 2 * t + 1 >= g : g >= 2 * t + 1};
#pragma unroll 1
    for (int c = 0; c < blocks; ++c) {
      const int rows = min(C, seg_rows - c * C), s = c % STAGES;
      if (!wait_bar(&bars.full[s], (c / STAGES) & 1, gone)) break;
      if (c > 0 && !wait_bar(&bars.vs_empty[h2], (c - 1) & 1, gone)) break;
      tc::fence_after_sync();
      const uint32_t vt = tc::smem_u32(smem) + s * S::STAGE + 2 * S::KB;
      __nv_bfloat162 chk = __floats2bfloat162_rn(0.f, 0.f);
      auto decay = [&](auto tag) {
        constexpr int N = decltype(tag)::value;
#pragma unroll
        for (int x = 0; x < 2; ++x) {  // 16 tokens each
          float f[2][2];  // of tokens 2t (+ 1), + 8
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const int j = h2 * 32 + x * 16 + (y >> 1) * 8 + 2 * t + (y & 1), at = rev ? C - 1 - j : j;
            f[y >> 1][y & 1] = at < rows ? P.u * pw[max(rows - 1 - at + P.e, 0)] : 0.f;
          }
#pragma unroll
          for (int z = 0; z < 2; ++z) {  // 16 value rows each
            const int col = w * 32 + z * 16;
            uint32_t u[4], o[4][N];
            mma::ldsm4t(u, vt + (col >> 6) * 8192 + swz(h2 * 32 + x * 16 + (m >> 1) * 8 + r8, ((col & 63) >> 3) + (m & 1)));
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              chk = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&u[y]), __floats2bfloat162_rn(0.f, 0.f), chk);
              decayed<N>(u[y], f[y >> 1][0], f[y >> 1][1], o[y]);
            }
#pragma unroll
            for (int p = 0; p < N; ++p)
              tmem_st_frag(lanes + (static_cast<uint32_t>(z * 16) << 16) + S::F + 32 * p + h2 * 16 + x * 8, o[0][p], o[1][p],
                           o[2][p], o[3][p]);
          }
        }
      };
      if (w * 32 < DV) {
        if (parts == 3)
          decay(std::integral_constant<int, 3>{});
        else
          decay(std::integral_constant<int, 2>{});
        if (__low2float(chk) != 0.f || __high2float(chk) != 0.f)  // NaN too
          *static_cast<volatile int*>(&bad_s[s]) = c + 1;
        tc::tmem_wait_st();
      }
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&bars.vs_full[h2]);
        if (!STATE_ONLY) mbar_arrive(&bars.noted[s]);
      }
      if (!STATE_ONLY && h2) {
        const int b = c & 1;
        if (c > 1 && !wait_bar(&bars.p_empty[b], ((c >> 1) - 1) & 1, gone)) break;
        if (!wait_bar(&bars.sc_full, c & 1, gone)) break;
        tc::fence_after_sync();
        const uint32_t pt = tc::smem_u32(smem) + S::P_OFF + b * S::PB;
        float v[8], next[8];
        tmem_ld_frag(my, next);
#pragma unroll 1
        for (int n = 0; n < 8; n += 2) {
          tmem_wait_ld(next);
#pragma unroll
          for (int x = 0; x < 8; ++x) v[x] = next[x];
          if (n < 6) {
            tmem_ld_frag(my + 8 * n + 16, next);
          } else {
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.sc_empty);
          }
          uint32_t o[2][2];
#pragma unroll
          for (int z = 0; z < 2; ++z)
#pragma unroll
            for (int y = 0; y < 2; ++y) {  // columns of group n + z, rows g + 8 y: group number 2 w + y
              const int away = rev ? n + z - 2 * w - y : 2 * w + y - n - z;  // the same for the whole warp
              float a = v[4 * z + 2 * y], d = v[4 * z + 2 * y + 1];
              if (away > 0) {
                const float f = P.a * pw[8 * away - 8];
                a *= f * edge[0];
                d *= f * edge[1];
              } else {  // selects, not products with 0: masked scores may be Inf or NaN
                a = away == 0 && see[0] ? a * own[0] : 0.f;
                d = away == 0 && see[1] ? d * own[1] : 0.f;
              }
              o[z][y] = mma::pack2(a, d);
            }
          // matrices (rows 8 y, columns 8 n)
          stsm4(pt + swz(16 * w + 8 * (m & 1) + r8, n + (m >> 1)), o[0][0], o[0][1], o[1][0], o[1][1]);
        }
        tc::fence_smem_to_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.p_full[b]);
      }
    }
  } else {
    regs_dec<48>();
    if (warp == 16) {  // ------------------------------------------------------- the copies
      const CUtensorMap* const maps[3] = {&M.map[M.m[blockIdx.z][0]], &M.map[M.m[blockIdx.z][1]],
                                          &M.map[M.m[blockIdx.z][2]]};
      const int hq = h / P.qg, hk = h / P.kg, hv = h / P.vg;
      int sent = 0;
#pragma unroll 1
      for (int c = 0; c < blocks; ++c) {
        const int rows = min(C, seg_rows - c * C), s = c % STAGES;
        if (c >= STAGES && !wait_bar(&bars.empty[s], ((c / STAGES) - 1) & 1, gone)) break;
        const int64_t row = first + down * c;
        const uint32_t base = tc::smem_u32(smem) + s * S::STAGE;
        sent = c + 1;
        uint64_t* const bar = rows == C ? &bars.full[s] : &bars.part;
        if (tc::elect_one()) {
          constexpr int BOXES = (STATE_ONLY ? 1 : 2) * (DK / 64) + DV / 64;
          mbar_expect(bar, BOXES * 8192);
          const int r = static_cast<int>(row);
#pragma unroll
          for (int hf = 0; hf < DK / 64; ++hf) {
            if (!STATE_ONLY) tma_box(base + hf * 8192, maps[0], hf * 64, r, hq, bi, bar);
            tma_box(base + S::KB + hf * 8192, maps[1], hf * 64, r, hk, bi, bar);
          }
#pragma unroll
          for (int hf = 0; hf < DV / 64; ++hf) tma_box(base + 2 * S::KB + hf * 8192, maps[2], hf * 64, r, hv, bi, bar);
        }
        __syncwarp();
        if (rows != C) {
          // The last block's rows that are not in the sequence, another one's or none's, become zeros in k and v:
          // they may hold Inf or NaN.  (Those of q give outputs that are not stored.)
          if (!tc::mbar_wait(&bars.part, 0, 0, 10000)) {
            *gone = 1;
            break;
          }
          const int lo = rev ? 0 : rows, n = C - rows;
          char* const kv = smem + s * S::STAGE + S::KB;
#pragma unroll 1
          for (int x = lane; x < n * 8; x += 32)
#pragma unroll
            for (int hf = 0; hf < (DK + DV) / 64; ++hf)
              *reinterpret_cast<uint4*>(kv + hf * 8192 + lo * 128 + x * 16) = make_uint4(0, 0, 0, 0);
          tc::fence_smem_to_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars.full[s]);
        }
      }
      // no copy is left in flight, whatever made the roles leave
      for (int c = max(0, sent - STAGES); c < sent; ++c) tc::mbar_wait(&bars.full[c % STAGES], (c / STAGES) & 1, 0, 10000);
    } else if (warp == 19 && tc::elect_one()) {  // -------------------- the sums U, from one thread
      const uint32_t base = desc_lo(tc::smem_u32(smem));  // descriptors count in units of 16 bytes
      constexpr uint32_t d_u = idesc_bf16(128, DK, false, true);
      bool ok = true;
#pragma unroll 1
      for (int c = 0; ok && (c + 1 < blocks || (keep_last && c < blocks)); ++c) {
        const uint32_t k = base + ((c % STAGES) * S::STAGE + S::KB) / 16;
        if (!(ok = wait_one(&bars.u_empty, c & 1, gone))) break;
#pragma unroll
        for (int h2 = 0; h2 < 2; ++h2) {  // the tokens' halves, as the decayed values come
          if (!(ok = ok && wait_one(&bars.vs_full[h2], c & 1, gone))) break;
          tc::fence_after_sync();
          const uint32_t a = tm + S::F + h2 * 16, b = k + h2 * 256;
          // the small parts first
          if (parts == 3) {
            mma_ts(tm + S::U, a + 64, b, d_u, h2 > 0);
            mma_ts(tm + S::U, a + 72, b + 128, d_u, 1);
          }
          mma_ts(tm + S::U, a + 32, b, d_u, parts == 3 || h2 > 0);
          mma_ts(tm + S::U, a + 40, b + 128, d_u, 1);
          mma_ts(tm + S::U, a, b, d_u, 1);
          mma_ts(tm + S::U, a + 8, b + 128, d_u, 1);
          tc::mma_commit(&bars.vs_empty[h2]);
          if (h2) tc::mma_commit(&bars.u_full);
        }
      }
    } else if (!STATE_ONLY && warp == 18 && tc::elect_one()) {  // ----- the scores and outputs, from another
      const uint32_t base = desc_lo(tc::smem_u32(smem));
      const int kd16 = (P.kd + 15) / 16;
      constexpr uint32_t d_sc = idesc_bf16(64, 64, false, false), d_o1 = idesc_bf16(128, 64, false, false),
                         d_o2 = idesc_bf16(128, 64, true, false);
      auto scores = [&](int c) {
        const uint32_t q = base + (c % STAGES) * (S::STAGE / 16), k = q + S::KB / 16;
        if (!wait_one(&bars.full[c % STAGES], (c / STAGES) & 1, gone)) return false;
        if (c > 0 && !wait_one(&bars.sc_empty, (c - 1) & 1, gone)) return false;
        tc::fence_after_sync();
#pragma unroll
        for (int x = 0; x < DK / 16; ++x) {
          const uint32_t off = (x >> 2) * 512 + (x & 3) * 2;
          if (x < kd16) mma_ss(tm + S::SC, q + off, k + off, d_sc, x > 0);
        }
        tc::mma_commit(&bars.sc_full);
        return true;
      };
      bool ok = blocks == 0 || scores(0);
#pragma unroll 1
      for (int c = 0; ok && c < blocks; ++c) {
        const int b = c & 1;
        const uint32_t q = base + (c % STAGES) * (S::STAGE / 16), v = q + 2 * S::KB / 16;
        if (!(ok = wait_one(&bars.s_full, c & 1, gone))) break;
        if (c > 0 && !(ok = wait_one(&bars.o_empty, (c - 1) & 1, gone))) break;
        tc::fence_after_sync();
#pragma unroll
        for (int x = 0; x < DK / 16; ++x)
          if (x < kd16) mma_ts(tm + S::O, tm + S::S + x * 8, q + (x >> 2) * 512 + (x & 3) * 2, d_o1, x > 0);
        tc::mma_commit(&bars.s_empty);
        if (!(ok = wait_one(&bars.p_full[b], (c >> 1) & 1, gone))) break;
        tc::fence_after_sync();
        const uint32_t p = base + (S::P_OFF + b * S::PB) / 16;
#pragma unroll
        for (int x = 0; x < C / 16; ++x) mma_ss(tm + S::O + 64, v + x * 128, p + x * 2, d_o2, x > 0);
        tc::mma_commit(&bars.o_full);
        if (c + 1 < blocks && !(ok = scores(c + 1))) break;
      }
    }
  }
  __syncwarp();
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  if (warp == 19) tc::tmem_dealloc(tm, 512);
  if (tid == 0 && gone_s != 0 && status != nullptr) atomicOr_system(status, TTC_STATUS_MMA_TIMEOUT);
}

}  // namespace da
}  // namespace ttc
