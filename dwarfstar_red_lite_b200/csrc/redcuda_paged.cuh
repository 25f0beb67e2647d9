// Layout of the decode attention over a paged cache (redcuda_paged.cu).
#pragma once
#include "redcuda_vals.cuh"

namespace rc {

// Warps and stages of a block, blocks of a multiprocessor: twelve stages of 16 KB an SM in every form. Six warps x two stages x one block: two documents of 131072 and some 115000 positions 86 us, 64 ragged
// sequences 22, 238 of 147 positions 42, 205 of up to 33 36; three x two x two 89, 20, 35, 24 (one block's head begins or ends while the other's tiles flow); two x three x two 90, 21, 36, 25;
// two x two x three 93, 21, 34, 22.
constexpr int KV_WARPS = 3, KV_STAGES = 2, KV_BLOCKS = 2;
constexpr uint32_t KV_HEAD_COST = 12u;           // what a head's begin and end take, in tiles
constexpr uint32_t KV_MIN_TILES = 3u;            // tiles that a block takes at least: one a warp

struct AttendArgs {
    void *k, *v;
    uint64_t page_stride, token_stride, head_stride;     // in elements
    const int32_t *table, *lens;
    const void *q, *k_new, *v_new;
    uint64_t q_stride, new_stride;
    void *out;
    float *lse, *part, *part_ml;
    uint32_t *meta, *status;
    uint32_t table_width, page_size, n_pages, n_seqs, n_kv, n_q, G, gsplit;     // G: query heads of a K/V head, in gsplit groups of 8
    float scale_log2;
};

// A tile: 8 KB of K rows, then 8 KB of V rows, the 16-byte pieces of a row turned by its number so that eight rows' pieces of one column lie in
// different banks.
template <class T, int HD> struct KvTile {
    static constexpr uint32_t ROW = HD * sizeof(T), TP = 8192u / ROW, CPR = ROW / 16u, BYTES = 2u * 8192u;
    static constexpr int TPL = TP > 32u ? 2 : 1;         // rows that a lane looks up
    static_assert(TP * CPR % 32u == 0u && TP >= 8u && TP <= 64u && CPR >= 8u, "tile");
    static __device__ __forceinline__ uint32_t swizzle(uint32_t row, uint32_t c) { return c ^ (row & 7u); }
};

}  // namespace rc
