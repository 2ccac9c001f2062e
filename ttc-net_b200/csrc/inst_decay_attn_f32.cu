#include "decay_attn_f32.cuh"
#include "decay_attn_launch.cuh"

namespace ttc {
namespace da {

template <int DK, int DV, bool STATE_ONLY>
int launch_f32_shape(const Args& A, int passes, cudaStream_t st) {
  using S = F32Shape<DK, DV, STATE_ONLY>;
  auto k = decay_attn_f32_kernel<DK, DV, STATE_ONLY>;
  cudaError_t e = cudaSuccess;
  if (S::SMEM > 48 * 1024) e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
  if (e == cudaSuccess) {
    const unsigned x = static_cast<unsigned>(A.items) + clearing_ctas(A, STATE_ONLY);
    k<<<dim3(x, static_cast<unsigned>(A.H), static_cast<unsigned>(passes)), kF32Threads, S::SMEM, st>>>(A);
    e = cudaGetLastError();
  }
  if (e == cudaSuccess) return TTC_OK;
  char buf[256];
  snprintf(buf, sizeof(buf), "decay_attn_f32_kernel launch: %s", cudaGetErrorString(e));
  return set_error(TTC_ERR_CUDA, buf);
}

int launch_f32(const Args& A, int passes, bool state_only, cudaStream_t st) {
  const int kd = width_class_f32(A.pass[0].kd), vd = width_class_f32(A.pass[0].vd);
#define TTC_DA(K, V)   \
  if (kd == K && vd == V) \
  return state_only ? launch_f32_shape<K, V, true>(A, passes, st) : launch_f32_shape<K, V, false>(A, passes, st)
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

}  // namespace da
}  // namespace ttc
