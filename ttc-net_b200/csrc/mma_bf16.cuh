// Warp-level bf16 matrix products (mma.sync m16n8k16, fp32 accumulators) and what feeds them:
// ldmatrix, the swizzled shared-memory tile and the split of an fp32 value into bf16 parts.
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>

namespace ttc {
namespace mma {

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// Four 8x8 matrices of 16-bit values; lane 8 m + r gives the address of row r of matrix m.
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// d += a b; a: 16 x 16 row-major fragment, b: 16 x 8 column-major fragment (two registers).
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float lo_f(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float hi_f(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }

// What is left of x after its bf16 part p: exact, and 0 where p is not finite (Inf - Inf would
// turn an infinity into NaN plus NaN).
__device__ __forceinline__ float rest(float x, float p) {
  const float r = x - p;
  return fabsf(r) <= 3.0e38f ? r : 0.f;
}

// (x, y) as NS bf16 parts each, largest first: the sum of three parts holds 24 bits.
template <int NS>
__device__ __forceinline__ void split2(float x, float y, uint32_t (&p)[NS]) {
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    p[s] = pack2(x, y);
    if (s + 1 < NS) {
      x = rest(x, lo_f(p[s]));
      y = rest(y, hi_f(p[s]));
    }
  }
}

// Byte offset of the 16-byte piece `c` of row `r` in a tile of COLS 16-bit columns.  The piece
// index is xor-ed with the row so that the 8 rows of an 8x8 matrix fall in 8 different bank
// groups, whichever way they are read.
template <int COLS>
__device__ __forceinline__ uint32_t tile_off(int r, int c) {
  if constexpr (COLS == 32) {
    return static_cast<uint32_t>(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
  } else {
    return static_cast<uint32_t>(r * (COLS * 2) + ((c ^ (r & 7)) << 4));
  }
}

}  // namespace mma
}  // namespace ttc
