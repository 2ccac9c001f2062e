#include "decay_attn_launch.cuh"
#include "decay_attn_tc.cuh"

namespace ttc {
namespace da {

template <int DK, int DV, bool STATE_ONLY>
int launch_tc_shape(const Args& A, int passes, int* status, cudaStream_t st) {
  auto k = decay_attn_tc_kernel<DK, DV, STATE_ONLY>;
  const int smem = TcShape<DK, DV>::smem(A.parts);
  // the warpgroups' register shares (192 + 96 + 3 x 64) are taken from what the CTA is launched with
  cudaFuncAttributes at;
  cudaError_t e = cudaFuncGetAttributes(&at, k);
  if (e == cudaSuccess && at.numRegs < 96)
    return set_error(TTC_ERR_UNSUPPORTED, "decay_attn_tc_kernel: built with fewer than 96 registers a thread");
  if (e == cudaSuccess) e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess) {
    const unsigned x = static_cast<unsigned>(A.items) + (!STATE_ONLY && A.cu != nullptr ? 1u : 0u);
    k<<<dim3(x, static_cast<unsigned>(A.H), static_cast<unsigned>(passes)), kTcThreads, smem, st>>>(A, status);
    e = cudaGetLastError();
  }
  if (e == cudaSuccess) return TTC_OK;
  char buf[256];
  snprintf(buf, sizeof(buf), "decay_attn_tc_kernel launch: %s", cudaGetErrorString(e));
  return set_error(TTC_ERR_CUDA, buf);
}

int launch_bf16(const Args& A, int passes, bool state_only, bool tc, int* status, cudaStream_t st) {
  if (!tc) return launch<1>(A, passes, state_only, st);
  const bool wide_k = A.pass[0].kd > 64, wide_v = A.pass[0].vd > 64;
#define TTC_TC(K, V)                                                                   \
  return state_only ? launch_tc_shape<K, V, true>(A, passes, status, st) : launch_tc_shape<K, V, false>(A, passes, status, st)
  if (wide_k && wide_v) TTC_TC(128, 128);
  if (wide_k) TTC_TC(128, 64);
  if (wide_v) TTC_TC(64, 128);
  TTC_TC(64, 64);
#undef TTC_TC
}

}  // namespace da
}  // namespace ttc
