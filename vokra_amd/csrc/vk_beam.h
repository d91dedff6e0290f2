// vk_beam.h — launcher of beam search's selection (vk_beam.hip). The C-ABI layer
// (vk_beam_capi.hip) checks its arguments.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

constexpr int kBeamMost = 32;      // beams of a group
constexpr int kBeamOut = 64;       // continuations of a group
constexpr int kBeamSlice = 4096;   // columns of the smaller slices at most (the workspace is sized by them)

struct BeamStat {
    double sum;  // of e^(x - max) over the slice
    float max;
    int count;   // its best columns that are listed
};

struct BeamArgs {
    const float* logits;
    size_t stride;  // floats from row to row
    const float* scores;
    const int* ended;  // NULL: none has
    float* out_scores;
    int *out_parents, *out_tokens, *out_ended;  // out_ended NULL: not written
    unsigned long long* keys;  // [row][slice][n_out]
    BeamStat* stats;           // [row][slice]
    int groups, beams, vocab, n_out, end_token;
    int slices, width, group;  // set by the launcher: slices of a row, their columns, threads of a group
};

namespace vk {
// slices, width and group are filled in here
hipError_t launch_beam_select(hipStream_t s, BeamArgs a);
}  // namespace vk
