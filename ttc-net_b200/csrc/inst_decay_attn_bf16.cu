#include "decay_attn_launch.cuh"
namespace ttc {
namespace da {
int launch_bf16(const Args& A, int passes, bool state_only, cudaStream_t st) { return launch<1>(A, passes, state_only, st); }
}  // namespace da
}  // namespace ttc
