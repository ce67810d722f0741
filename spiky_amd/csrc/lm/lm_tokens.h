// lm_tokens.h -- launchers of the operators of include/spiky_lm_tokens.h.
//
// Internal to libspiky_lut.so.
#pragma once

#include "../../../include/spiky_lm_tokens.h"
#include "lm_kernels.h"

namespace spiky {
namespace lm {

hipError_t launch_embed(const spiky_lm_embed_args &a, void *out, hipStream_t st);
uint64_t embed_workspace(const spiky_lm_embed_args &a);
hipError_t launch_embed_backward(const spiky_lm_embed_args &a, const void *d_out, int64_t d_out_stride, void *d_weight,
                                 void *workspace, hipStream_t st);

uint64_t beam_select_workspace(const spiky_lm_beams_args &a);
hipError_t launch_beam_select(const spiky_lm_beams_args &a, void *workspace, hipStream_t st);

hipError_t launch_reorder(const spiky_lm_state *states, uint64_t count, const void *parents, bool parents_i64,
                          uint64_t searches, uint64_t beams, uint64_t n, hipStream_t st);

}  // namespace lm
}  // namespace spiky
