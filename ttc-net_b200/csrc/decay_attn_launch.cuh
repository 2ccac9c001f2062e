// Launches of the attention with a decay, one translation unit for each element type.
#pragma once

#include <cstdio>

#include "decay_attn.cuh"
#include "ttc_b200.h"

namespace ttc {
int set_error(int code, const char* msg);

namespace da {

// Compiled tile widths: a head dim runs in the next one, its missing columns zeros.
inline int width_class_f32(int d) { return d <= 32 ? 32 : (d <= 64 ? 64 : 128); }
inline int width_class_bf16(int d) { return d <= 64 ? 64 : 128; }

// CTAs of a head, behind its items, that clear the rows behind the last packed sequence: how many rows these are is
// known on the device only.  One for every 8192 rows of the whole, so that none has more than these to clear and those
// with nothing to do stay few beside the rows' own (24 prompts in 9 600 rows: two a head, 135 us against 134 with one).
inline unsigned clearing_ctas(const Args& A, bool state_only) {
  return state_only || A.cu == nullptr ? 0u : 1u + static_cast<unsigned>(A.T / 8192);
}

// All passes of `A` have the same width classes.
int launch_bf16(const Args& A, int passes, bool state_only, int* status, cudaStream_t st);
int launch_f32(const Args& A, int passes, bool state_only, cudaStream_t st);

}  // namespace da
}  // namespace ttc
