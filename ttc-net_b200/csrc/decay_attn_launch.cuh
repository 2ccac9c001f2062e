// Launch of decay_attn_kernel for one element type; one translation unit instantiates each.
#pragma once

#include <cstdio>

#include "decay_attn.cuh"
#include "ttc_b200.h"

namespace ttc {
int set_error(int code, const char* msg);

namespace da {

// Compiled tile widths: a head dim runs in the next one, its missing columns zeros.
inline int width_class(int d) { return d <= 32 ? 32 : (d <= 64 ? 64 : 128); }

template <int DK, int DV, int NP, bool STATE_ONLY>
int launch_shape(const Args& A, int passes, cudaStream_t st) {
  using S = Shape<DK, DV, NP, STATE_ONLY>;
  auto k = decay_attn_kernel<DK, DV, NP, STATE_ONLY>;
  cudaError_t e = cudaSuccess;
  if (S::SMEM > 48 * 1024) e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
  if (e == cudaSuccess) {
    // packed rows: one more CTA a head for the rows behind the last sequence
    const unsigned x = static_cast<unsigned>(A.items) + (!STATE_ONLY && A.cu != nullptr ? 1u : 0u);
    k<<<dim3(x, static_cast<unsigned>(A.H), static_cast<unsigned>(passes)), S::THREADS, S::SMEM, st>>>(A);
    e = cudaGetLastError();
  }
  if (e == cudaSuccess) return TTC_OK;
  char buf[256];
  snprintf(buf, sizeof(buf), "decay_attn_kernel launch: %s", cudaGetErrorString(e));
  return set_error(TTC_ERR_CUDA, buf);
}

// All passes of `A` have the same width classes.
template <int NP>
int launch(const Args& A, int passes, bool state_only, cudaStream_t st) {
  const int kd = width_class(A.pass[0].kd), vd = width_class(A.pass[0].vd);
#define TTC_DA(K, V)                                            \
  if (kd == K && vd == V)                                       \
  return state_only ? launch_shape<K, V, NP, true>(A, passes, st) : launch_shape<K, V, NP, false>(A, passes, st)
  TTC_DA(32, 32);
  TTC_DA(32, 64);
  TTC_DA(32, 128);
  TTC_DA(64, 32);
  TTC_DA(64, 64);
  TTC_DA(64, 128);
  TTC_DA(128, 32);
  TTC_DA(128, 64);
  TTC_DA(128, 128);
#undef TTC_DA
  return set_error(TTC_ERR_UNSUPPORTED, "decay_attn: no kernel for these head dims");
}

// bf16: `tc` picks the tcgen05 kernel (decay_attn_tc.cuh), else the warp-level one.
int launch_bf16(const Args& A, int passes, bool state_only, bool tc, int* status, cudaStream_t st);
int launch_f32(const Args& A, int passes, bool state_only, cudaStream_t st);

}  // namespace da
}  // namespace ttc
