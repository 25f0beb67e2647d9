// Arguments of the gated delta rule's kernels (redcuda_delta.cu).
#pragma once
#include "redcuda_vals.cuh"

namespace rc {

constexpr int DELTA_WARPS = 4, DELTA_ROWS = 32;          // a block: 32 rows of one head's state

struct DeltaArgs {
    const void *q, *k, *v;
    uint64_t q_stride, k_stride, v_stride;               // elements between two tokens
    const float *gate, *beta;
    float *state;
    void *out;
    const int32_t *cu, *slots;
    uint32_t *status;
    uint32_t n_tokens, n_slots, groups, rank, first_seq;
    float scale;
};

}  // namespace rc
