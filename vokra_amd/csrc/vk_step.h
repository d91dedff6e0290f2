// vk_step.h — launchers of the operators around a decode step that are no
// part of a session: rotary positions by a plan (vk_rope.hip) and the rules
// that logits pass before the greedy choice (vk_rules.hip). The C-ABI layer
// (vk_step_capi.hip) checks their arguments.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

struct RopeArgs {
    const float *q, *k;
    float *q_out, *k_out;
    size_t q_stride, k_stride, qo_stride, ko_stride;  // floats from row to row
    const int* positions;
    const uint64_t* turn;  // [rot / 2] fraction of a turn per position, in 2^-64
    float mag;
    int rows, heads_q, heads_k, hd, rot;
    int units, head_lanes;  // set by the launcher
};

// A context's workspace of the greedy choice: rows' maxima, then their counters.
constexpr int kRulesRows = 65536;
constexpr size_t kRulesPartBytes = (size_t)kRulesRows * 12;

struct RulesArgs {
    const float* logits;
    float* out;      // NULL: not written
    int* next;       // NULL: not chosen
    size_t stride;   // floats from row to row, of logits and out
    const int *hist, *hist_off, *bias_ids, *bias_off;
    const float *repetition, *presence, *frequency, *bias;
    const uint32_t* mask;
    size_t mask_stride;
    unsigned long long* best;  // zero between calls
    unsigned* done;            // zero between calls
    int rows, vocab, n_hist, n_bias;
};

namespace vk {
// units and head_lanes are filled in here
hipError_t launch_rope_turn(hipStream_t s, RopeArgs a, bool pairs);
hipError_t launch_rules_clear(hipStream_t s, void* part);
hipError_t launch_rules(hipStream_t s, const RulesArgs& a);
}  // namespace vk
