#include "decay_attn_launch.cuh"
#include "decay_attn_tc.cuh"

namespace ttc {
namespace da {

namespace {

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
  static const EncodeTiled f = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return f;
}

int encode_map(EncodeTiled encode, CUtensorMap* map, const void* p, const int64_t* s, int heads, int dim, int64_t T,
               int64_t batch) {
  // a dimension of one element may have any stride; 16 bytes are the least that is allowed
  const auto bytes = [](int64_t size, int64_t stride) { return static_cast<cuuint64_t>(size == 1 ? 16 : stride * 2); };
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(dim), static_cast<cuuint64_t>(T), static_cast<cuuint64_t>(heads),
                              static_cast<cuuint64_t>(batch)};
  const cuuint64_t strides[3] = {bytes(T, s[1]), bytes(heads, s[2]), bytes(batch, s[0])};
  const cuuint32_t box[4] = {64, C, 1, 1}, one[4] = {1, 1, 1, 1};
  const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(p), dims, strides, box, one,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r == CUDA_SUCCESS) return TTC_OK;
  char buf[128];
  snprintf(buf, sizeof(buf), "decay_attn: cuTensorMapEncodeTiled returned %d", static_cast<int>(r));
  return set_error(TTC_ERR_CUDA, buf);
}

// The maps of the passes' operands, one for each tensor (at most four: q, k, v and the output's gradient).
int make_maps(const Args& A, int passes, TcMaps& M) {
  if (A.T == 0) return TTC_OK;  // nothing is read
  // the driver's call wants a current context, which a thread that only made runtime calls may lack
  // (autograd's backward threads): cudaSetDevice makes the device's own current
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaSetDevice(dev) != cudaSuccess)
    return set_error(TTC_ERR_CUDA, "decay_attn: no current device");
  const EncodeTiled encode = encode_tiled();
  if (encode == nullptr) return set_error(TTC_ERR_CUDA, "decay_attn: the driver has no cuTensorMapEncodeTiled");
  struct Key {
    const void* p;
    int64_t s[3];
    int heads, dim;
  } seen[4];
  int n = 0;
  const int64_t batch = A.cu ? 1 : A.n_seq;
  for (int i = 0; i < passes; ++i) {
    const Pass& P = A.pass[i];
    const Key use[3] = {{P.q, {P.qs[0], P.qs[1], P.qs[2]}, A.H / P.qg, P.kd},
                        {P.k, {P.ks[0], P.ks[1], P.ks[2]}, A.H / P.kg, P.kd},
                        {P.v, {P.vs[0], P.vs[1], P.vs[2]}, A.H / P.vg, P.vd}};
    for (int j = 0; j < 3; ++j) {
      const Key& u = use[j];
      int at = 0;
      while (at < n && !(seen[at].p == u.p && seen[at].s[0] == u.s[0] && seen[at].s[1] == u.s[1] &&
                         seen[at].s[2] == u.s[2] && seen[at].heads == u.heads && seen[at].dim == u.dim))
        ++at;
      M.m[i][j] = at;
      if (at < n) continue;
      if (n == 4) return set_error(TTC_ERR_INVALID, "decay_attn: more than four operands");
      seen[n++] = u;
      if (int rc = encode_map(encode, &M.map[at], u.p, u.s, u.heads, u.dim, A.T, batch)) return rc;
    }
    if (!P.o_f32) {
      const int64_t os[3] = {A.T * A.H * P.vd, static_cast<int64_t>(A.H) * P.vd, P.vd};
      if (int rc = encode_map(encode, &M.out[i], P.o, os, A.H, P.vd, A.T, batch)) return rc;
    }
  }
  return TTC_OK;
}

}  // namespace

template <int DK, int DV, bool STATE_ONLY>
int launch_tc_shape(const Args& A, int passes, int* status, cudaStream_t st) {
  auto k = decay_attn_tc_kernel<DK, DV, STATE_ONLY>;
  constexpr int smem = TcShape<DK, DV>::SMEM;
  TcMaps M{};
  if (int rc = make_maps(A, passes, M)) return rc;
  // the warpgroups' register shares (192 + 96 + 72 + 72 + 48) are taken from what the CTA is launched with
  cudaFuncAttributes at;
  cudaError_t e = cudaFuncGetAttributes(&at, k);
  if (e == cudaSuccess && at.numRegs < 96)
    return set_error(TTC_ERR_UNSUPPORTED, "decay_attn_tc_kernel: built with fewer than 96 registers a thread");
  if (e == cudaSuccess) e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess) {
    const unsigned x = static_cast<unsigned>(A.items) + clearing_ctas(A, STATE_ONLY);
    k<<<dim3(x, static_cast<unsigned>(A.H), static_cast<unsigned>(passes)), kTcThreads, smem, st>>>(A, M, status);
    e = cudaGetLastError();
  }
  if (e == cudaSuccess) return TTC_OK;
  char buf[256];
  snprintf(buf, sizeof(buf), "decay_attn_tc_kernel launch: %s", cudaGetErrorString(e));
  return set_error(TTC_ERR_CUDA, buf);
}

int launch_bf16(const Args& A, int passes, bool state_only, int* status, cudaStream_t st) {
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
