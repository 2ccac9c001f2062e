#include "decay_attn_launch.cuh"
namespace ttc {
namespace da {
int launch_f32(const Args& A, int passes, bool state_only, cudaStream_t st) { return launch<3>(A, passes, state_only, st); }
}  // namespace da
}  // namespace ttc
