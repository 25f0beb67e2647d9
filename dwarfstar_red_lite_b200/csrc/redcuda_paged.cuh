// Layout of the decode attention over a paged cache (redcuda_paged.cu).
#pragma once
#include "redcuda_vals.cuh"

namespace rc {

// Warps and stages of a block, blocks of a multiprocessor: twelve stages of 16 KB an SM in every form. Six warps x two stages x one block: two documents of 131072 and some 115000 positions 86 us, 64 ragged
// sequences 22, 238 of 147 positions 42, 205 of up to 33 36; three x two x two 89, 20, 35, 24 (one block's head begins or ends while the other's tiles flow); two x three x two 90, 21, 36, 25;
// two x two x three 93, 21, 34, 22.
// Caches of floats with heads of up to 128 have the registers for twelve warps an SM, which wait less for one another's tiles: tiles of 8 KB and twice the blocks. us, 16 KB x two blocks -> 8 KB x four: heads of 128, 32 over 8, 24 sequences
// of 500 to 1999 positions 48.8 -> 45.7, 64 of up to 2048 42.8 -> 32.5, 200 of up to 40 31 -> 23, 4 of 30000 to 60000 242 -> 234; 64 over 8 76 -> 60; heads of 64, 8 over 8 37.9 -> 29.5.
// 16-bit caches with heads of 128 lose by the same what they gain: 200 of up to 40 28 -> 22, 64 of up to 2048 24.2 -> 22.6, 1 of 8000 12.8 -> 14.8, 24 of 500 to 1999 26.5 -> 28.1.
constexpr int KV_WARPS = 3, KV_STAGES = 2, KV_BLOCKS = 2;
constexpr uint32_t KV_HEAD_COST = 12u;           // what a head's begin and end take, in tiles
constexpr uint32_t KV_MIN_TILES = 3u;            // tiles that a block takes at least: one a warp

// A cluster of blocks a head: how many blocks, for how many heads at most, and up to how many tiles a warp can have (by the page table's width) for 16-bit caches and caches of floats. us, dealt out -> in clusters:
// F16, 2 K/V heads of 256: 1 sequence of 50 positions 10.5 -> 7.8, of 613 11.1 -> 9.3, of 1500 12.5 -> 11.7; 4 of 613 12.9 -> 9.9; 9 of 613 14.2 -> 11.0; 18 of 300 15.1 -> 15.8. BF16, 8 of 128: 1 of 613 9.7 -> 6.0,
// 4 of 613 10.8 -> 6.8. F32, 2 of 256: 1 of 200 12.4 -> 9.9, of 613 11.6 -> 13.6; 4 of 100 12.8 -> 7.8.
constexpr uint32_t KV_CLUSTER = 8u, KV_CLUSTER_HEADS = 32u, KV_CLUSTER_TILES = 4u, KV_CLUSTER_TILES_F32 = 2u;

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
    uint32_t clusters;                                   // heads, where each has a cluster of blocks; 0: the form that deals tiles out
    float scale_log2;
};

// A tile: 8 KB (or 4) of K rows, then as much of V rows, the 16-byte pieces of a row turned by its number so that eight rows' pieces of one column lie in
// different banks.
constexpr uint32_t kv_half(uint32_t size, uint32_t hd) { return size == 4u && hd <= 128u ? 4096u : 8192u; }
constexpr uint32_t kv_blocks(uint32_t size, uint32_t hd) { return KV_BLOCKS * (8192u / kv_half(size, hd)); }
template <class T, int HD> struct KvTile {
    static constexpr uint32_t HALF = kv_half(sizeof(T), HD), ROW = HD * sizeof(T), TP = HALF / ROW, CPR = ROW / 16u, BYTES = 2u * HALF;
    static constexpr int TPL = TP > 32u ? 2 : 1;         // rows that a lane looks up
    static_assert(TP * CPR % 32u == 0u && TP >= 8u && TP <= 64u && CPR >= 8u, "tile");
    static __device__ __forceinline__ uint32_t swizzle(uint32_t row, uint32_t c) { return c ^ (row & 7u); }
};

}  // namespace rc
