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

// whole prompts with states of 128 in chunks on the tensor cores (redcuda_delta_chunk.cu)
uint64_t delta_chunk_workspace(uint32_t type, uint32_t groups, uint32_t rank, uint32_t n_tokens, uint32_t n_seqs);
int launch_delta_chunks(const DeltaArgs &A, uint32_t type, uint32_t n_seqs, uint8_t *ws, cudaStream_t s);

#ifdef __CUDACC__
// The state slot of sequence b, or -1: none, out of range, or one that an earlier sequence has (two sequences would write it at once).
// For the whole block (it meets a barrier).
__device__ __forceinline__ int32_t delta_slot(const int32_t *slots, uint32_t n_slots, uint32_t b, uint32_t *status) {
    if (!slots) return b < n_slots ? (int32_t)b : -1;
    const int32_t s = slots[b];
    bool bad = s < -1 || (s >= 0 && (uint32_t)s >= n_slots);
    if (s >= 0) for (uint32_t i = threadIdx.x; i < b; i += blockDim.x) bad |= slots[i] == s;
    bad = __syncthreads_or(bad);
    if (bad && threadIdx.x == 0u && status) status[ST_SLOT] = 1u;
    return bad ? -1 : s;
}
#endif

}  // namespace rc
