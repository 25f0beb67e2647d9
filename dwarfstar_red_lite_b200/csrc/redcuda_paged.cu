// A paged K/V cache: rows of prompts written to its pages, and attention of one new token per sequence over them.
//
//   k_kv_append     a warp per token: its K and V rows, converted, to the page that the table names
//   k_kv_attend     decode attention over the sequences' whole lengths (below)
//   k_kv_attend_join  sums the parts of sequences that several blocks worked on
//   k_kv_attend_cluster  the same for few heads of moderate length, in one launch
#include "redcuda_paged.cuh"
#include "redcuda_stage.cuh"
#include "../../include/redcuda.h"

#include <cooperative_groups.h>
#include <math.h>
#include <type_traits>

namespace rc {

namespace cg = cooperative_groups;

struct AppendArgs {
    void *k, *v;
    uint64_t page_stride, token_stride, head_stride;
    const int32_t *table, *start, *cu;
    const void *k_new, *v_new;
    uint64_t row_stride;
    uint32_t table_width, page_size, n_pages, n_seqs, n_tokens, n_kv, hd;
    uint32_t *status;
};

// What bounds it is the copy: a row read once, written once (30011 tokens of 32 prompts, 2 heads of 256, BF16: 123 MB in 21 us, 5.9 TB/s; 500 tokens 2.5 us, a launch). A lane moves VEC values (16 bytes of the cache's type) of K and of V at a time.
template <class C, class R>
__global__ void __launch_bounds__(128) k_kv_append(AppendArgs A) {
    pdl_prologue();
    constexpr int VEC = 16 / sizeof(C), PART = 16 / sizeof(R) < VEC ? 16 / sizeof(R) : VEC;
    const uint32_t lane = threadIdx.x & 31u, t = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (A.cu && A.status)                        // a thread looks at every so many-th sequence's bounds
        for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < A.n_seqs; i += (uint64_t)gridDim.x * blockDim.x)       // up to 2^36 threads
            if (!seq_bounds(A.cu, (uint32_t)i, A.n_tokens)) A.status[ST_SEQ_BOUNDS] = 1u;
    if (t >= A.n_tokens) return;
    uint32_t b = t, at = 0u;
    if (A.cu) {
        b = find_seq(A.cu, A.n_seqs, t, A.n_tokens);
        if (b >= A.n_seqs) return;               // of no sequence
        at = t - (uint32_t)A.cu[b];
    }
    const int32_t s = A.start[b];
    if (s < 0) return;
    const uint64_t pos = (uint64_t)(uint32_t)s + at, pi = pos / A.page_size;
    const int32_t page = pi < A.table_width ? A.table[(uint64_t)b * A.table_width + pi] : -1;
    if (page < 0 || (uint32_t)page >= A.n_pages) { if (A.status && lane == 0u) A.status[ST_PAGE_RANGE] = 1u; return; }
    const uint64_t dst = (uint64_t)page * A.page_stride + (pos - pi * A.page_size) * A.token_stride, src = (uint64_t)t * A.row_stride;
    const uint32_t n = A.n_kv * A.hd;
#pragma unroll 2
    for (uint32_t i = lane * VEC; i < n; i += 32u * VEC) {
        const uint32_t h = i / A.hd;
        const uint64_t d = dst + (uint64_t)h * A.head_stride + (i - h * A.hd);
        float x[VEC / PART][PART], y[VEC / PART][PART];
#pragma unroll
        for (int p = 0; p < VEC / PART; ++p) {
            load_vals<PART>(reinterpret_cast<const R *>(A.k_new) + src + i + p * PART, x[p]);
            load_vals<PART>(reinterpret_cast<const R *>(A.v_new) + src + i + p * PART, y[p]);
        }
        store_vals<VEC>(reinterpret_cast<C *>(A.k) + d, *reinterpret_cast<float (*)[VEC]>(&x[0][0]));
        store_vals<VEC>(reinterpret_cast<C *>(A.v) + d, *reinterpret_cast<float (*)[VEC]>(&y[0][0]));
    }
}

template <class C, class R> static int launch_append(const AppendArgs &A, cudaStream_t s) {
    RC_LAUNCH((k_kv_append<C, R>), (A.n_tokens + 3u) / 4u, 128, 0, s, A);
    RC_LAUNCHED();
    return 1;
}
template <class C> static int launch_append_rows(const AppendArgs &A, uint32_t in_type, cudaStream_t s) {
    return in_type == VT_F32 ? launch_append<C, float>(A, s) : in_type == VT_F16 ? launch_append<C, __half>(A, s) : launch_append<C, __nv_bfloat16>(A, s);
}

// ---- decode attention -------------------------------------------------------------------------------------------------------
// With x_p = scale log2(e) q . k_p, a part of the positions is summed up as m = max x_p, l = sum 2^(x_p - m), O = sum 2^(x_p - m) v_p; parts are joined
// by rescaling to the common m, and out = O / l.
//
// What bounds it is the cache's bytes (504 MB of two long documents: 89 us, 5.6 TB/s; 77 us at the measured copy rate) and, for short sequences, the beginning and end of each head (some 3 us
// a block: lengths, page table, queries, rows, each a read that waits for the one before).
// The work is cut by bytes: a tile is 16 KB (8 of some caches of floats) of K and V of one K/V head, all tiles of all (sequence, K/V head, group of 8 query heads) are
// counted through in that order, and every block takes an equal run of them, whatever the lengths are: they are read on the device, so that a
// captured call follows them. A head costs as much as some tiles more (KV_HEAD_COST). A run that begins or ends inside a sequence's head leaves (m, l, O) in the workspace, at most two of them a
// block, for k_kv_attend_join; what a block has whole it writes itself. A warp has a ring of tiles of its own, so that the warps of a block meet only where a head ends.

__device__ __forceinline__ float kv_lse(float m, float l) { return l == 0.f ? -INFINITY : m * 0.693147180559945309f + logf(l); }

// the positions of sequence b that can be attended to
__device__ __forceinline__ uint32_t kv_len(const AttendArgs &A, uint32_t b) {
    const int32_t n = A.lens[b];
    const uint64_t most = (uint64_t)A.table_width * A.page_size;
    return n <= 0 ? 0u : (uint64_t)(uint32_t)n > most ? (uint32_t)most : (uint32_t)n;
}

// What a head counts in the deal: its tiles, and as many more as its begin and end take (KV_HEAD_COST). Those come first: a run that ends among them leaves
// the whole head to the next block.
template <class L> __device__ __forceinline__ uint32_t kv_cost(uint32_t len) { return len ? (len + L::TP - 1u) / L::TP + KV_HEAD_COST : 0u; }

// One tile of a warp's ring: its rows requested, rows beyond the end or without a page as zeros. Returns the rows that count, as bits.
template <class T, int HD>
__device__ __forceinline__ uint64_t kv_request(const AttendArgs &A, uint32_t b, uint32_t kvh, uint32_t len, uint32_t tile, uint32_t dst) {
    using L = KvTile<T, HD>;
    const uint32_t lane = threadIdx.x & 31u;
    int64_t off[L::TPL];
    uint64_t valid = 0;
#pragma unroll
    for (int j = 0; j < L::TPL; ++j) {
        const uint32_t r = j * 32u + lane, pos = tile * L::TP + r;
        off[j] = -1;
        if (r < L::TP && pos < len) {
            const uint32_t pi = pos / A.page_size;
            const int32_t page = A.table[(uint64_t)b * A.table_width + pi];
            if (page >= 0 && (uint32_t)page < A.n_pages)
                off[j] = (int64_t)((uint64_t)page * A.page_stride + (uint64_t)(pos - pi * A.page_size) * A.token_stride + (uint64_t)kvh * A.head_stride);
            else if (A.status) A.status[ST_PAGE_RANGE] = 1u;
        }
        valid |= (uint64_t)__ballot_sync(0xffffffffu, off[j] >= 0) << (32 * j);
    }
    const T *kb = reinterpret_cast<const T *>(A.k), *vb = reinterpret_cast<const T *>(A.v);
#pragma unroll
    for (int i = 0; i < (int)(L::TP * L::CPR / 32u); ++i) {
        const uint32_t n = i * 32u + lane, row = n / L::CPR, c = n % L::CPR;
        const int64_t o = __shfl_sync(0xffffffffu, off[(i * 32 / (int)L::CPR) / 32], (int)(row & 31u));
        const uint32_t sz = o >= 0 ? 16u : 0u, to = dst + row * L::ROW + L::swizzle(row, c) * 16u;
        const uint64_t src = (uint64_t)(o >= 0 ? o : 0) + c * (16u / sizeof(T));
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(to), "l"(kb + src), "r"(sz) : "memory");
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(to + L::TP * L::ROW), "l"(vb + src), "r"(sz) : "memory");
    }
    return valid;
}

// A warp's share of a part: every KV_WARPS-th tile of [t0, t1), up to NH query heads; (m, l, O) to shared memory. For a cache of floats the sums on CUDA cores, 32 / NH positions at a time:
// their 32 scores are summed over the lanes together and end in a lane each. A position costs a warp 4 NH instructions for its products and some 20 for the rest (packed fp32), where the bytes of a position of 128 leave
// an SM 23 cycles; hence the form for 4 heads. With it no pipe is the bound: 24 sequences of 500 to 1999 positions, 32 heads over 8 of 128, 45.7 us: issue slots 44 %, fp32 pipe 29 %, DRAM 61 % of nominal, and the
// warps' first stall is on global memory (the next tile of a ring of two).
template <class T, class QT, int HD, int NH>
__device__ __forceinline__ void attend_part_f32(const AttendArgs &A, uint32_t b, uint32_t kvh, uint32_t h0, uint32_t nh, uint32_t len, uint32_t t0, uint32_t t1,
                                            uint8_t *ring, uint64_t *valid, float *p_sh, float *m_out, float *l_out, float *o_out) {
    using L = KvTile<T, HD>;
    constexpr int E = HD / 32, PS = 32 / NH;
    static_assert(L::TP % PS == 0, "whole steps");
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint32_t ring_s = (uint32_t)__cvta_generic_to_shared(ring);
    // element i of a lane: a 16-byte piece (or less) of the row, two pieces for rows of 1 KB
    auto elem = [&](int i) { return E * sizeof(T) > 16 ? (uint32_t)(i / 4) * 128u + lane * 4u + (uint32_t)(i % 4) : lane * E + (uint32_t)i; };
    float2 q[NH][E / 2], o[NH][E / 2];
    const QT *qp = reinterpret_cast<const QT *>(A.q) + (uint64_t)b * A.q_stride + (uint64_t)h0 * HD;
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int i = 0; i < E; i += 2) {
            q[h][i / 2] = make_float2(0.f, 0.f);
            if (h < (int)nh) q[h][i / 2] = make_float2(to_f32(qp[h * HD + elem(i)]) * A.scale_log2, to_f32(qp[h * HD + elem(i + 1)]) * A.scale_log2);
            o[h][i / 2] = make_float2(0.f, 0.f);
        }
    float m = -INFINITY, l = 0.f;                // of head lane / PS; l: this lane's share
    uint32_t next = t0 + warp;
#pragma unroll 1
    for (int s = 0; s < KV_STAGES - 1; ++s) {
        if (next < t1) { const uint64_t w = kv_request<T, HD>(A, b, kvh, len, next, ring_s + s * L::BYTES); if (lane == 0u) valid[s] = w; }
        asm volatile("cp.async.commit_group;" ::: "memory");
        next += KV_WARPS;
    }
    uint32_t st = 0;
    for (uint32_t t = t0 + warp; t < t1; t += KV_WARPS) {
        const uint32_t fill = st == 0u ? KV_STAGES - 1 : st - 1u;
        asm volatile("cp.async.wait_group %0;" :: "n"(KV_STAGES - 2) : "memory");
        __syncwarp();
        if (next < t1) { const uint64_t w = kv_request<T, HD>(A, b, kvh, len, next, ring_s + fill * L::BYTES); if (lane == 0u) valid[fill] = w; }
        asm volatile("cp.async.commit_group;" ::: "memory");
        next += KV_WARPS;
        const uint64_t live = valid[st];
        const uint8_t *kt = ring + st * L::BYTES, *vt = kt + L::TP * L::ROW;
        auto row = [&](const uint8_t *base, uint32_t r, float2 (&x)[E / 2]) {
#pragma unroll
            for (int i = 0; i < E; i += (E * sizeof(T) > 16 ? 4 : E)) {
                constexpr int N = E * sizeof(T) > 16 ? 4 : E;
                const uint32_t byte = elem(i) * sizeof(T);
                float y[N];
                load_vals<N>(reinterpret_cast<const T *>(base + r * L::ROW + L::swizzle(r, byte / 16u) * 16u + byte % 16u), y);
#pragma unroll
                for (int j = 0; j < N; j += 2) x[(i + j) / 2] = make_float2(y[j], y[j + 1]);
            }
        };
#pragma unroll 1
        for (uint32_t r = 0; r < L::TP; r += PS) {
            const uint32_t bits = (uint32_t)(live >> r) & ((1u << PS) - 1u);
            if (!bits) continue;
            float s[32];                         // score of head i / PS, position r + i % PS: this lane's part
#pragma unroll
            for (int j = 0; j < PS; ++j) {
                float2 k[E / 2];
                row(kt, r + j, k);
#pragma unroll
                for (int h = 0; h < NH; ++h) {
                    float2 a = __fmul2_rn(q[h][0], k[0]);
#pragma unroll
                    for (int i = 1; i < E / 2; ++i) a = __ffma2_rn(q[h][i], k[i], a);
                    s[h * PS + j] = a.x + a.y;
                }
            }
            // 32 sums over 32 lanes: each exchange halves the values that a lane carries; value i ends in lane i
#pragma unroll
            for (int w = 16; w; w >>= 1) {
                const bool hi = lane & w;
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (i < w) {
                        const float keep = hi ? s[w + i] : s[i], send = hi ? s[i] : s[w + i];
                        s[i] = keep + __shfl_xor_sync(0xffffffffu, send, w);
                    }
            }
            const float x = (bits >> (lane % PS)) & 1u ? s[0] : -INFINITY;
            float mx = x;
#pragma unroll
            for (int w = 1; w < PS; w <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
            const float mn = fmaxf(m, mx), base = mn == -INFINITY ? 0.f : mn, alpha = exp2f(m - base), p = exp2f(x - base);
            const bool moved = __any_sync(0xffffffffu, mn > m);
            m = mn;
            l = l * alpha + p;
            __syncwarp();
            p_sh[lane] = p;
            if (lane % PS == 0u) p_sh[32u + lane / PS] = alpha;
            __syncwarp();
            if (moved) {
#pragma unroll
                for (int h = 0; h < NH; ++h) {
                    const float a = p_sh[32 + h];
#pragma unroll
                    for (int i = 0; i < E / 2; ++i) o[h][i] = __fmul2_rn(o[h][i], make_float2(a, a));
                }
            }
#pragma unroll
            for (int k = 0; k < PS; k += 4) {
                float2 v[4][E / 2];
#pragma unroll
                for (int j = 0; j < 4; ++j) row(vt, r + k + j, v[j]);
#pragma unroll
                for (int h = 0; h < NH; ++h) {
                    const float4 p4 = *reinterpret_cast<const float4 *>(p_sh + h * PS + k);
#pragma unroll
                    for (int i = 0; i < E / 2; ++i) {
                        o[h][i] = __ffma2_rn(make_float2(p4.x, p4.x), v[0][i], o[h][i]);
                        o[h][i] = __ffma2_rn(make_float2(p4.y, p4.y), v[1][i], o[h][i]);
                        o[h][i] = __ffma2_rn(make_float2(p4.z, p4.z), v[2][i], o[h][i]);
                        o[h][i] = __ffma2_rn(make_float2(p4.w, p4.w), v[3][i], o[h][i]);
                    }
                }
            }
        }
        __syncwarp();
        st = st + 1u == KV_STAGES ? 0u : st + 1u;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
    for (int w = 1; w < PS; w <<= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
    if (lane % PS == 0u) { m_out[lane / PS] = m; l_out[lane / PS] = l; }
    if (NH < 8 && lane < 8u - NH) { m_out[NH + lane] = -INFINITY; l_out[NH + lane] = 0.f; }
    __syncthreads();                             // the rings are read no more
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int i = 0; i < E; i += 2) { o_out[h * HD + elem(i)] = o[h][i / 2].x; o_out[h * HD + elem(i + 1)] = o[h][i / 2].y; }
}

// The same share on the tensor cores, for a cache of 16-bit values. m16n8k16 has 16 rows where a group has 8 heads: rows 0-7 carry the upper digit of the
// heads' queries (or weights), rows 8-15 the lower, so that two digits cost what one would, and the two halves of an accumulator (both in the same
// lane) are added at the end. A query of floats over F16 is q 2^e = hi + lo with 2^e such that the head's largest is below 2^15 (22 bits); a query of the
// cache's own type is its upper digit. A weight is 2^(x - m) = hi + lo likewise, 22 bits in F16 (with m chosen KV_P_BIAS lower, so that small weights keep
// their lower digit), 16 in BF16, where the output is rounded to 8. m is moved only when the maximum has grown by more than KV_SLACK, as
// that rescales the accumulators; the weights stay below 2^(KV_P_BIAS + KV_SLACK).
constexpr float KV_P_BIAS = 6.f, KV_SLACK = 8.f;

template <class T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t *>(&h); }
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) { const __nv_bfloat162 h = __floats2bfloat162_rn(a, b); return *reinterpret_cast<const uint32_t *>(&h); }
template <class T> __device__ __forceinline__ float2 unpack2(uint32_t x);
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t x) { return __half22float2(*reinterpret_cast<const __half2 *>(&x)); }
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t x) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&x)); }
template <class T> __device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

template <class T, class QT, int HD>
__device__ __forceinline__ void attend_part_mma(const AttendArgs &A, uint32_t b, uint32_t kvh, uint32_t h0, uint32_t nh, uint32_t len, uint32_t t0, uint32_t t1,
                                            uint8_t *ring, uint64_t *valid, float *m_out, float *l_out, float *o_out) {
    using L = KvTile<T, HD>;
    constexpr bool TWO = !std::is_same<T, QT>::value;
    constexpr float BIAS = std::is_same<T, __half>::value ? KV_P_BIAS : 0.f;
    constexpr int KS = HD / 16, NT = L::TP / 8, DT = HD / 8;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, g = lane >> 2, c2 = (lane & 3u) * 2u;
    const uint32_t ring_s = (uint32_t)__cvta_generic_to_shared(ring);
    uint32_t next = t0 + warp;
#pragma unroll 1
    for (int s = 0; s < KV_STAGES - 1; ++s) {
        if (next < t1) { const uint64_t w = kv_request<T, HD>(A, b, kvh, len, next, ring_s + s * L::BYTES); if (lane == 0u) valid[s] = w; }
        asm volatile("cp.async.commit_group;" ::: "memory");
        next += KV_WARPS;
    }
    uint32_t st = 0;
    // the query of head g: elements 16 s + c2, + 1, + 8, + 9 of it
    uint32_t qh[KS][2], ql[TWO ? KS : 1][2];
    float sc = A.scale_log2;
    {
        const QT *qp = reinterpret_cast<const QT *>(A.q) + (uint64_t)b * A.q_stride + (uint64_t)(h0 + g) * HD;
        const bool have = g < nh;
        if constexpr (TWO) {
            float most = 0.f;
            if (have)
#pragma unroll
                for (int s = 0; s < KS; ++s)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const float2 x = *reinterpret_cast<const float2 *>(qp + 16 * s + c2 + 8 * u);
                        most = fmaxf(most, fmaxf(fabsf(x.x), fabsf(x.y)));
                    }
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
            int e = 0;
            if (most > 0.f && most < INFINITY) e = min(141 - (int)(__float_as_uint(most) >> 23), 126);       // 127 + 14: the largest in [2^14, 2^15)
            const float up = __uint_as_float((uint32_t)(127 + e) << 23);
            sc *= 1.f / up;
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    float2 x = make_float2(0.f, 0.f);
                    if (have) x = *reinterpret_cast<const float2 *>(qp + 16 * s + c2 + 8 * u);
                    x.x *= up; x.y *= up;
                    qh[s][u] = pack2<T>(x.x, x.y);
                    const float2 h = unpack2<T>(qh[s][u]);
                    ql[s][u] = pack2<T>(x.x - h.x, x.y - h.y);
                }
        } else {
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int u = 0; u < 2; ++u) qh[s][u] = have ? *reinterpret_cast<const uint32_t *>(qp + 16 * s + c2 + 8 * u) : 0u;
        }
    }
    float o[DT][4], m = -INFINITY, l = 0.f;      // m, l: of head g; l this lane's share
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[d][i] = 0.f;
    // what a lane addresses of four 8 x 8 pieces: K rows lane % 8 and pieces lane / 8; V rows (lane / 8 % 2) * 8 + lane % 8 and pieces lane / 16
    const uint32_t kr = lane & 7u, kc = lane >> 3, vr = (lane >> 3 & 1u) * 8u + (lane & 7u), vc = lane >> 4;
    for (uint32_t t = t0 + warp; t < t1; t += KV_WARPS) {
        const uint32_t fill = st == 0u ? KV_STAGES - 1 : st - 1u;
        asm volatile("cp.async.wait_group %0;" :: "n"(KV_STAGES - 2) : "memory");
        __syncwarp();
        if (next < t1) { const uint64_t w = kv_request<T, HD>(A, b, kvh, len, next, ring_s + fill * L::BYTES); if (lane == 0u) valid[fill] = w; }
        asm volatile("cp.async.commit_group;" ::: "memory");
        next += KV_WARPS;
        const uint64_t live = valid[st];
        const uint32_t kt = ring_s + st * L::BYTES, vt = kt + L::TP * L::ROW;
        float x[NT][2];
#pragma unroll
        for (int n = 0; n < NT; n += 2) {        // two runs of eight positions, each in two sums
            float c[4][4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) c[i][j] = 0.f;
#pragma unroll
            for (int s = 0; s < KS; s += 2) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t row = (uint32_t)(n + i) * 8u + kr;
                    uint32_t k[4];
                    ldsm4(k, kt + row * L::ROW + L::swizzle(row, (uint32_t)s * 2u + kc) * 16u);
                    mma16816<T>(c[2 * i], qh[s][0], TWO ? ql[TWO ? s : 0][0] : 0u, qh[s][1], TWO ? ql[TWO ? s : 0][1] : 0u, k[0], k[1]);
                    mma16816<T>(c[2 * i + 1], qh[s + 1][0], TWO ? ql[TWO ? s + 1 : 0][0] : 0u, qh[s + 1][1], TWO ? ql[TWO ? s + 1 : 0][1] : 0u, k[2], k[3]);
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float v = TWO ? (c[2 * i][j] + c[2 * i + 1][j]) + (c[2 * i][j + 2] + c[2 * i + 1][j + 2]) : c[2 * i][j] + c[2 * i + 1][j];
                    const uint32_t pos = (uint32_t)(n + i) * 8u + c2 + (uint32_t)j;
                    x[n + i][j] = (live >> pos) & 1u ? v * sc : -INFINITY;
                }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int n = 0; n < NT; ++n) mx = fmaxf(mx, fmaxf(x[n][0], x[n][1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const bool move = mx > m + KV_SLACK;     // from -infinity too
        if (__any_sync(0xffffffffu, move)) {
            const float to = move ? mx : m, alpha = move ? exp2f(m - to) : 1.f;
            m = to;
            l *= alpha;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[d][i] *= alpha;
        }
        const float base = m == -INFINITY ? 0.f : m - BIAS;
        uint32_t pa[NT / 2][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float p0 = exp2f(x[n][0] - base), p1 = exp2f(x[n][1] - base);
            l += p0 + p1;
            const uint32_t hi = pack2<T>(p0, p1);
            const float2 h = unpack2<T>(hi);
            pa[n / 2][(n & 1) * 2] = hi;
            pa[n / 2][(n & 1) * 2 + 1] = pack2<T>(p0 - h.x, p1 - h.y);
        }
#pragma unroll
        for (int j = 0; j < NT / 2; ++j)
#pragma unroll
            for (int d = 0; d < DT; d += 2) {
                const uint32_t row = (uint32_t)j * 16u + vr;
                uint32_t v[4];
                ldsm4_t(v, vt + row * L::ROW + L::swizzle(row, (uint32_t)d + vc) * 16u);
                mma16816<T>(o[d], pa[j][0], pa[j][1], pa[j][2], pa[j][3], v[0], v[1]);
                mma16816<T>(o[d + 1], pa[j][0], pa[j][1], pa[j][2], pa[j][3], v[2], v[3]);
            }
        __syncwarp();
        st = st + 1u == KV_STAGES ? 0u : st + 1u;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if ((lane & 3u) == 0u) { m_out[g] = m - BIAS; l_out[g] = l; }
    __syncthreads();                             // the rings are read no more
#pragma unroll
    for (int d = 0; d < DT; ++d) *reinterpret_cast<float2 *>(o_out + g * HD + d * 8u + c2) = make_float2(o[d][0] + o[d][2], o[d][1] + o[d][3]);
}

// the new row of sequence b, K/V head kvh, to its page (the whole block)
template <class T, class QT, int HD>
__device__ __forceinline__ void kv_write_new(const AttendArgs &A, uint32_t b, uint32_t kvh, uint32_t pos) {
    const uint32_t pi = pos / A.page_size;
    const int32_t page = A.table[(uint64_t)b * A.table_width + pi];
    if (page < 0 || (uint32_t)page >= A.n_pages) return;       // reported where the row is read
    const uint64_t d = (uint64_t)page * A.page_stride + (uint64_t)(pos - pi * A.page_size) * A.token_stride + (uint64_t)kvh * A.head_stride;
    const uint64_t s = (uint64_t)b * A.new_stride + (uint64_t)kvh * HD;
    for (uint32_t i = threadIdx.x; i < 2u * HD; i += blockDim.x) {
        const uint32_t e = i % HD;
        const QT *from = reinterpret_cast<const QT *>(i < HD ? A.k_new : A.v_new);
        reinterpret_cast<T *>(i < HD ? A.k : A.v)[d + e] = from_f32<T>(to_f32(from[s + e]));
    }
}

// NH: heads that a group can have (4 only for a cache of floats)
// Over 16-bit caches it takes all 255 registers, and with heads of 64 and 256 spills 36 to 56 bytes a thread; over floats with heads of 128 and eight query heads 168, and 36 bytes.
template <class T, class QT, int HD, int NH>
__global__ void __launch_bounds__(KV_WARPS * 32, kv_blocks(sizeof(T), HD)) k_kv_attend(AttendArgs A) {
    pdl_prologue();
    using L = KvTile<T, HD>;
    extern __shared__ __align__(128) uint8_t sm[];
    __shared__ uint64_t s_sum[KV_WARPS], s_base, s_valid[KV_WARPS][KV_STAGES];
    __shared__ uint32_t s_b;
    __shared__ __align__(16) float s_p[sizeof(T) == 4 ? KV_WARPS : 1][40], s_m[KV_WARPS][8], s_l[KV_WARPS][8], s_scale[8];
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, HG = A.n_kv * A.gsplit;
    QT *const out = reinterpret_cast<QT *>(A.out);

    // how many tiles there are, and the sequence in which this block's run begins
    const uint32_t per = (A.n_seqs + KV_WARPS * 32u - 1u) / (KV_WARPS * 32u), b_lo = min(A.n_seqs, tid * per), b_hi = min(A.n_seqs, b_lo + per);
    uint64_t mine = 0;
    for (uint32_t b = b_lo; b < b_hi; ++b) mine += kv_cost<L>(kv_len(A, b));
    uint64_t incl = mine;
#pragma unroll
    for (int w = 1; w < 32; w <<= 1) { const uint64_t x = __shfl_up_sync(0xffffffffu, incl, w); if (lane >= (uint32_t)w) incl += x; }
    if (lane == 31u) s_sum[warp] = incl;
    __syncthreads();
    uint64_t total = 0;
    for (uint32_t w = 0; w < KV_WARPS; ++w) { if (w < warp) incl += s_sum[w]; total += s_sum[w]; }
    total *= HG;
    const uint64_t q = max((total + gridDim.x - 1u) / gridDim.x, (uint64_t)KV_MIN_TILES), u0 = q * blockIdx.x, u1 = min(total, u0 + q);
    uint64_t base = (incl - mine) * HG;
    if (u0 < u1 && base <= u0 && u0 < incl * HG) {
        uint32_t b = b_lo;
        for (;; ++b) { const uint64_t n = (uint64_t)kv_cost<L>(kv_len(A, b)) * HG; if (u0 < base + n) break; base += n; }
        s_b = b; s_base = base;
    }
    for (uint32_t b = blockIdx.x; b < A.n_seqs; b += gridDim.x) {
        if (A.status && tid == 0u && A.lens[b] > 0 && (uint32_t)A.lens[b] != kv_len(A, b)) A.status[ST_PAGE_RANGE] = 1u;
        if (kv_len(A, b) == 0u) {                // nothing to attend to
            for (uint32_t i = tid; i < A.n_q * HD; i += KV_WARPS * 32u) out[(uint64_t)b * A.n_q * HD + i] = from_f32<QT>(0.f);
            if (A.lse) for (uint32_t i = tid; i < A.n_q; i += KV_WARPS * 32u) A.lse[(uint64_t)b * A.n_q + i] = -INFINITY;
        }
    }
    __syncthreads();
    uint32_t parts_b = 0, parts_h = 0, parts_n = 0;            // the head that begins here and ends in a later block
    if (u0 < u1) {
        uint32_t b = s_b;
        base = s_base;
        uint64_t u = u0;
        while (u < u1) {
            const uint32_t len = kv_len(A, b), nt = (len + L::TP - 1u) / L::TP, cost = kv_cost<L>(len);
            if (u >= base + (uint64_t)cost * HG) { base += (uint64_t)cost * HG; ++b; continue; }
            const uint32_t hg = (uint32_t)((u - base) / cost);
            const uint64_t end = base + (uint64_t)(hg + 1u) * cost;             // of this head; its tiles are the last nt units before it
            const uint32_t t0 = end - u >= nt ? 0u : nt - (uint32_t)(end - u), t1 = end <= u1 ? nt : end - u1 >= nt ? 0u : nt - (uint32_t)(end - u1);
            u = min(end, u1);
            if (t0 == t1) continue;              // the run ends inside the head's surcharge
            const uint32_t kvh = hg / A.gsplit, g0 = (hg % A.gsplit) * 8u, h0 = kvh * A.G + g0, nh = min(8u, A.G - g0);
            if (A.k_new && t1 == nt && len == (uint32_t)A.lens[b]) kv_write_new<T, QT, HD>(A, b, kvh, len - 1u);
            __syncthreads();                     // the new row is written; what the last head left in shared memory has been read
            float *o_sh = reinterpret_cast<float *>(sm);
            uint8_t *ring = sm + warp * KV_STAGES * L::BYTES;
            float *o_warp = o_sh + warp * 8u * HD;
            if constexpr (sizeof(T) == 4)
                attend_part_f32<T, QT, HD, NH>(A, b, kvh, h0, nh, len, t0, t1, ring, s_valid[warp], s_p[sizeof(T) == 4 ? warp : 0], s_m[warp], s_l[warp], o_warp);
            else
                attend_part_mma<T, QT, HD>(A, b, kvh, h0, nh, len, t0, t1, ring, s_valid[warp], s_m[warp], s_l[warp], o_warp);
            __syncthreads();
            // the warps' parts together
            const bool whole = t0 == 0u && t1 == nt;
            const uint32_t slot = blockIdx.x * 2u + (t0 == 0u ? 1u : 0u);
            if (tid < 8u) {
                float M = s_m[0][tid], lt = 0.f;
#pragma unroll
                for (uint32_t j = 1; j < KV_WARPS; ++j) M = fmaxf(M, s_m[j][tid]);
                const float z = M == -INFINITY ? 0.f : M;
#pragma unroll
                for (uint32_t j = 0; j < KV_WARPS; ++j) { const float w = exp2f(s_m[j][tid] - z); lt += w * s_l[j][tid]; s_m[j][tid] = w; }
                s_scale[tid] = whole ? lt == 0.f ? 0.f : 1.f / lt : 1.f;
                if (!whole) { A.part_ml[slot * 16u + tid] = M; A.part_ml[slot * 16u + 8u + tid] = lt; }
                else if (tid < nh && A.lse) A.lse[(uint64_t)b * A.n_q + h0 + tid] = kv_lse(M, lt);
            }
            __syncthreads();
            for (uint32_t i = tid * 4u; i < (uint32_t)NH * HD; i += KV_WARPS * 128u) {
                const uint32_t h = i / HD;
                float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (uint32_t j = 0; j < KV_WARPS; ++j) {
                    const float4 y = *reinterpret_cast<const float4 *>(o_sh + j * 8u * HD + i);
                    const float w = s_m[j][h];
                    x[0] += w * y.x; x[1] += w * y.y; x[2] += w * y.z; x[3] += w * y.w;
                }
                const float f = s_scale[h];
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = x[e] * f;
                if (!whole) store_vals<4>(A.part + (uint64_t)slot * 8u * HD + i, x);
                else if (h < nh) store_vals<4>(out + ((uint64_t)b * A.n_q + h0) * HD + i, x);
            }
            if (t0 == 0u && t1 < nt) { parts_b = b; parts_h = hg; parts_n = (uint32_t)((end - 1u) / q) - blockIdx.x; }
        }
    }
    if (tid == 0u) { A.meta[blockIdx.x * 4u] = parts_b; A.meta[blockIdx.x * 4u + 1u] = parts_h; A.meta[blockIdx.x * 4u + 2u] = parts_n; }
}

// Grid (blocks of k_kv_attend, 8 heads): the head that begins in block x, if it ends in a later one. HD / 4 threads have four values each, 1024 / HD such rows of
// threads every so many-th part; what bounds it is the chain of dependent reads, so the first parts are requested with the weights.
template <class QT, int HD>
__global__ void __launch_bounds__(256) k_kv_attend_join(AttendArgs A) {
    pdl_prologue();
    constexpr uint32_t COLS = HD / 4, ROWS = 256u / COLS, AHEAD = 8u;
    extern __shared__ float s_w[];               // a weight for every part
    __shared__ float s_max[8], s_sum[8];
    __shared__ __align__(16) float s_o[ROWS][HD];
    const uint32_t c = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, col = tid % COLS, row = tid / COLS;
    const uint4 meta = *reinterpret_cast<const uint4 *>(A.meta + c * 4u);
    const uint32_t n = meta.z;
    if (n == 0u) return;
    const uint32_t b = meta.x, hg = meta.y, g0 = (hg % A.gsplit) * 8u, head = (hg / A.gsplit) * A.G + g0 + h;
    if (g0 + h >= A.G) return;
    auto slot = [&](uint32_t p) { return p == 0u ? c * 2u + 1u : (c + p) * 2u; };
    auto part = [&](uint32_t p) { return *reinterpret_cast<const float4 *>(A.part + ((uint64_t)slot(p) * 8u + h) * HD + col * 4u); };
    float4 x[AHEAD];
#pragma unroll
    for (uint32_t i = 0; i < AHEAD; ++i) x[i] = row + i * ROWS <= n ? part(row + i * ROWS) : make_float4(0.f, 0.f, 0.f, 0.f);
    float M = -INFINITY, l = 0.f;
    for (uint32_t p = tid; p <= n; p += 256u) {  // a head can have as many parts as there are blocks: two or four an SM
        const float m = A.part_ml[slot(p) * 16u + h], lp = A.part_ml[slot(p) * 16u + 8u + h], to = fmaxf(M, m), z = to == -INFINITY ? 0.f : to;
        l = l * exp2f(M - z) + lp * exp2f(m - z);
        M = to;
        s_w[p] = m;
    }
    const float M0 = M;
    for (int w = 16; w; w >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, w));
    if ((tid & 31u) == 0u) s_max[tid >> 5] = M;
    __syncthreads();
    M = s_max[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) M = fmaxf(M, s_max[i]);
    const float z = M == -INFINITY ? 0.f : M;
    l *= exp2f(M0 - z);
    for (uint32_t p = tid; p <= n; p += 256u) s_w[p] = exp2f(s_w[p] - z);
    for (int w = 16; w; w >>= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
    if ((tid & 31u) == 0u) s_sum[tid >> 5] = l;
    __syncthreads();
    l = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) l += s_sum[i];
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](float w, float4 y) { o.x += w * y.x; o.y += w * y.y; o.z += w * y.z; o.w += w * y.w; };
#pragma unroll
    for (uint32_t i = 0; i < AHEAD; ++i)
        if (row + i * ROWS <= n) add(s_w[row + i * ROWS], x[i]);
#pragma unroll 8
    for (uint32_t p = row + AHEAD * ROWS; p <= n; p += ROWS) add(s_w[p], part(p));
    *reinterpret_cast<float4 *>(&s_o[row][col * 4u]) = o;
    __syncthreads();
    for (uint32_t i = tid; i < HD; i += 256u) {
        float sum = 0.f;
#pragma unroll
        for (uint32_t r = 0; r < ROWS; ++r) sum += s_o[r][i];
        reinterpret_cast<QT *>(A.out)[((uint64_t)b * A.n_q + head) * HD + i] = from_f32<QT>(l == 0.f ? 0.f : sum / l);
    }
    if (tid == 0u && A.lse) A.lse[(uint64_t)b * A.n_q + head] = kv_lse(M, l);
}

// ---- few heads of moderate length: one launch -----------------------------------------------------------------------------------------
// A cluster of eight blocks has a head, an eighth of its tiles each; their parts meet in shared memory, block r sums up query head r. What bounds it is the chain of reads; its figures stand at the rule (KV_CLUSTER_HEADS).
template <class T, class QT, int HD, int NH>
__global__ void __launch_bounds__(KV_WARPS * 32, kv_blocks(sizeof(T), HD)) k_kv_attend_cluster(AttendArgs A) {
    pdl_prologue();
    using L = KvTile<T, HD>;
    extern __shared__ __align__(128) uint8_t sm[];
    __shared__ uint64_t s_valid[KV_WARPS][KV_STAGES];
    __shared__ __align__(16) float s_p[sizeof(T) == 4 ? KV_WARPS : 1][40], s_m[KV_WARPS][8], s_l[KV_WARPS][8], s_part[2][8];
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t tid = threadIdx.x, warp = tid >> 5, rank = cluster.block_rank(), HG = A.n_kv * A.gsplit, b = blockIdx.x / KV_CLUSTER / HG, hg = blockIdx.x / KV_CLUSTER % HG;
    const uint32_t kvh = hg / A.gsplit, g0 = (hg % A.gsplit) * 8u, h0 = kvh * A.G + g0, nh = min(8u, A.G - g0);
    const uint32_t len = kv_len(A, b), nt = (len + L::TP - 1u) / L::TP, t0 = nt * rank / KV_CLUSTER, t1 = nt * (rank + 1u) / KV_CLUSTER;
    QT *const out = reinterpret_cast<QT *>(A.out) + ((uint64_t)b * A.n_q + h0) * HD;
    if (A.status && tid == 0u && rank == 0u && A.lens[b] > 0 && (uint32_t)A.lens[b] != len) A.status[ST_PAGE_RANGE] = 1u;
    if (len == 0u) {                             // nothing to attend to, for the whole cluster
        if (rank < nh) for (uint32_t i = tid; i < (uint32_t)HD; i += KV_WARPS * 32u) out[rank * HD + i] = from_f32<QT>(0.f);
        if (rank < nh && A.lse && tid == 0u) A.lse[(uint64_t)b * A.n_q + h0 + rank] = -INFINITY;
        return;
    }
    if (A.k_new && rank == KV_CLUSTER - 1u && len == (uint32_t)A.lens[b]) kv_write_new<T, QT, HD>(A, b, kvh, len - 1u);       // the last block has the last tile
    __syncthreads();
    float *o_sh = reinterpret_cast<float *>(sm);
    uint8_t *ring = sm + warp * KV_STAGES * L::BYTES;
    if constexpr (sizeof(T) == 4)
        attend_part_f32<T, QT, HD, NH>(A, b, kvh, h0, nh, len, t0, t1, ring, s_valid[warp], s_p[sizeof(T) == 4 ? warp : 0], s_m[warp], s_l[warp], o_sh + warp * 8u * HD);
    else
        attend_part_mma<T, QT, HD>(A, b, kvh, h0, nh, len, t0, t1, ring, s_valid[warp], s_m[warp], s_l[warp], o_sh + warp * 8u * HD);
    __syncthreads();
    if (tid < 8u) {
        float M = s_m[0][tid], lt = 0.f;
#pragma unroll
        for (uint32_t j = 1; j < KV_WARPS; ++j) M = fmaxf(M, s_m[j][tid]);
        const float z = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (uint32_t j = 0; j < KV_WARPS; ++j) { const float w = exp2f(s_m[j][tid] - z); lt += w * s_l[j][tid]; s_m[j][tid] = w; }
        s_part[0][tid] = M; s_part[1][tid] = lt;
    }
    __syncthreads();
    for (uint32_t i = tid * 4u; i < (uint32_t)NH * HD; i += KV_WARPS * 128u) {
        const uint32_t h = i / HD;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (uint32_t j = 0; j < KV_WARPS; ++j) {
            const float4 y = *reinterpret_cast<const float4 *>(o_sh + j * 8u * HD + i);
            const float w = s_m[j][h];
            x.x += w * y.x; x.y += w * y.y; x.z += w * y.z; x.w += w * y.w;
        }
        *reinterpret_cast<float4 *>(o_sh + i) = x;           // over the first warp's, which this thread alone reads
    }
    cluster.sync();
    if (rank < nh) {
        float M = -INFINITY, lt = 0.f, w[KV_CLUSTER];
#pragma unroll
        for (uint32_t r = 0; r < KV_CLUSTER; ++r) { w[r] = cluster.map_shared_rank(s_part[0], r)[rank]; M = fmaxf(M, w[r]); }
        const float z = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (uint32_t r = 0; r < KV_CLUSTER; ++r) { w[r] = exp2f(w[r] - z); lt += w[r] * cluster.map_shared_rank(s_part[1], r)[rank]; }
        for (uint32_t i = tid * 4u; i < (uint32_t)HD; i += KV_WARPS * 128u) {
            float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (uint32_t r = 0; r < KV_CLUSTER; ++r) {
                const float4 y = *reinterpret_cast<const float4 *>(cluster.map_shared_rank(o_sh, r) + rank * HD + i);
                x[0] += w[r] * y.x; x[1] += w[r] * y.y; x[2] += w[r] * y.z; x[3] += w[r] * y.w;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = lt == 0.f ? 0.f : x[e] / lt;
            store_vals<4>(out + rank * HD + i, x);
        }
        if (A.lse && tid == 0u) A.lse[(uint64_t)b * A.n_q + h0 + rank] = kv_lse(M, lt);
    }
    cluster.sync();                              // the others have read this block's shared memory
}

template <class T, class QT, int HD, int NH> static int launch_attend(const AttendArgs &A, uint32_t blocks, cudaStream_t s) {
    constexpr size_t smem = (size_t)KV_WARPS * KV_STAGES * KvTile<T, HD>::BYTES;
    static std::atomic<uint64_t> set{0};
    if (!raise_smem_limit(reinterpret_cast<const void *>(k_kv_attend<T, QT, HD, NH>), smem, set)) return 0;
    if (A.clusters) {
        static std::atomic<uint64_t> set_cluster{0};
        if (!raise_smem_limit(reinterpret_cast<const void *>(k_kv_attend_cluster<T, QT, HD, NH>), smem, set_cluster)) return 0;
        prof_begin("kv_attend", s);
        RC_LAUNCH_CLUSTER(KV_CLUSTER, (k_kv_attend_cluster<T, QT, HD, NH>), A.clusters * KV_CLUSTER, KV_WARPS * 32, smem, s, A);
        RC_LAUNCHED();
        prof_end(s);
        return 1;
    }
    prof_begin("kv_attend", s);
    RC_LAUNCH((k_kv_attend<T, QT, HD, NH>), blocks, KV_WARPS * 32, smem, s, A);
    RC_LAUNCHED();
    prof_end(s);
    prof_begin("kv_attend_join", s);
    RC_LAUNCH((k_kv_attend_join<QT, HD>), dim3(blocks, 8), 256, (blocks + 1u) * sizeof(float), s, A);
    RC_LAUNCHED();
    prof_end(s);
    return 1;
}
template <class T, class QT> static int launch_attend_hd(const AttendArgs &A, uint32_t hd, uint32_t blocks, cudaStream_t s) {
    if constexpr (sizeof(T) == 4)                // half the instructions where K/V heads have at most four query heads
        if (A.G <= 4u) return hd == 256u ? launch_attend<T, QT, 256, 4>(A, blocks, s) : hd == 128u ? launch_attend<T, QT, 128, 4>(A, blocks, s) : launch_attend<T, QT, 64, 4>(A, blocks, s);
    return hd == 256u ? launch_attend<T, QT, 256, 8>(A, blocks, s) : hd == 128u ? launch_attend<T, QT, 128, 8>(A, blocks, s) : launch_attend<T, QT, 64, 8>(A, blocks, s);
}

// the cache's strides in elements (0: dense), or a message
static int kv_check(const redcuda_paged_kv *kv, const char *who, uint64_t (&st)[3]) {
    RC_REQUIRE(kv && kv->k && kv->v, "%s: null cache", who);
    const uint32_t size = val_size(kv->type);
    RC_REQUIRE(size, "%s: cache type %u is none of F32, F16, BF16", who, kv->type);
    RC_REQUIRE(kv->head_dim == 64u || kv->head_dim == 128u || kv->head_dim == 256u, "%s: heads of %u values (64, 128 or 256 are served)", who, kv->head_dim);
    RC_REQUIRE(kv->n_kv && kv->n_kv <= 65535u && kv->page_size && kv->page_size <= 0x7fffffffu && kv->n_pages && kv->n_pages <= 0x7fffffffu, "%s: empty or too large cache", who);
    const bool dense = !kv->page_stride && !kv->token_stride && !kv->head_stride;
    st[2] = dense ? kv->head_dim : kv->head_stride;
    st[1] = dense ? (uint64_t)kv->n_kv * kv->head_dim : kv->token_stride;
    st[0] = dense ? st[1] * kv->page_size : kv->page_stride;
    for (int i = 0; i < 3; ++i)
        RC_REQUIRE(st[i] >= kv->head_dim && st[i] * size % 16u == 0u && st[i] < (1ull << 46), "%s: cache stride %llu (a multiple of 16 bytes, at least a head)", who, (unsigned long long)st[i]);
    RC_REQUIRE((uint64_t)kv->n_pages * st[0] < (1ull << 46), "%s: cache too large", who);
    RC_REQUIRE(aligned16(kv->k) && aligned16(kv->v), "%s: cache pointers are not 16-byte aligned", who);
    return 1;
}

// whether some array lies inside the cache
static bool kv_overlap(const redcuda_paged_kv *kv, const uint64_t (&st)[3], const void *p, uint64_t bytes) {
    const uint64_t n = ((uint64_t)(kv->n_pages - 1u) * st[0] + (uint64_t)(kv->page_size - 1u) * st[1] + (uint64_t)(kv->n_kv - 1u) * st[2] + kv->head_dim) * val_size(kv->type);
    return overlap(kv->k, n, p, bytes) || overlap(kv->v, n, p, bytes);
}
static uint64_t attend_workspace(uint32_t blocks, uint32_t hd) { return (uint64_t)blocks * (2u * (8u * hd + 16u) * 4u + 16u); }

}  // namespace rc

using namespace rc;

extern "C" {

int redcuda_kv_append_device(const redcuda_paged_kv *kv, const int32_t *table_dev, uint32_t table_width, uint32_t n_seqs, const int32_t *start_dev,
                             uint32_t n_tokens, const int32_t *cu_seqlens_dev, uint32_t in_type, const void *k_dev, const void *v_dev, uint64_t row_stride,
                             void *stream) {
    uint64_t st[3];
    if (!kv_check(kv, "kv append", st)) return 0;
    RC_REQUIRE(table_dev && start_dev && k_dev && v_dev && n_seqs && table_width, "kv append: null or empty argument");
    RC_REQUIRE(val_size(in_type), "kv append: rows of type %u (F32, F16 or BF16 are served)", in_type);
    RC_REQUIRE(n_seqs < 0x7fffffffu && n_tokens < 0x7fffffffu && table_width < 0x7fffffffu, "kv append: too many rows");
    RC_REQUIRE(cu_seqlens_dev || n_tokens == n_seqs, "kv append: %u rows for %u sequences without bounds", n_tokens, n_seqs);
    const uint64_t row = (uint64_t)kv->n_kv * kv->head_dim;
    if (!row_stride) row_stride = row;
    RC_REQUIRE(row_stride >= row && row_stride * val_size(in_type) % 16u == 0u && row_stride < (1ull << 32), "kv append: row stride %llu", (unsigned long long)row_stride);
    RC_REQUIRE(aligned16(k_dev) && aligned16(v_dev), "kv append: rows are not 16-byte aligned");
    RC_REQUIRE(aligned4(table_dev) && aligned4(start_dev) && aligned4(cu_seqlens_dev), "kv append: whole numbers are not 4-byte aligned");
    const uint64_t bytes = span_bytes(n_tokens, row_stride, row, val_size(in_type));
    RC_REQUIRE(!kv_overlap(kv, st, k_dev, bytes) && !kv_overlap(kv, st, v_dev, bytes), "kv append: the rows lie inside the cache");
    RC_REQUIRE(!kv_overlap(kv, st, table_dev, (uint64_t)n_seqs * table_width * 4u) && !kv_overlap(kv, st, start_dev, (uint64_t)n_seqs * 4u) && !kv_overlap(kv, st, cu_seqlens_dev, (n_seqs + 1ull) * 4u),
               "kv append: the page table, starts or bounds lie inside the cache");
    if (!require_device()) return 0;
    if (!n_tokens) return 1;
    AppendArgs A{kv->k, kv->v, st[0], st[1], st[2], table_dev, start_dev, cu_seqlens_dev, k_dev, v_dev, row_stride, table_width, kv->page_size, kv->n_pages, n_seqs, n_tokens, kv->n_kv,
                 kv->head_dim, status_words()};
    cudaStream_t s = (cudaStream_t)stream;
    prof_begin("kv_append", s);
    const int ok = kv->type == VT_F32 ? launch_append_rows<float>(A, in_type, s) : kv->type == VT_F16 ? launch_append_rows<__half>(A, in_type, s) : launch_append_rows<__nv_bfloat16>(A, in_type, s);
    prof_end(s);
    return ok;
}

uint64_t redcuda_kv_attend_workspace(const redcuda_paged_kv *kv, uint32_t n_q) {
    uint64_t st[3];
    if (!kv_check(kv, "kv attend", st)) return 0;
    RC_REQUIRE(n_q && n_q % kv->n_kv == 0u, "kv attend: %u query heads over %u K/V heads", n_q, kv->n_kv);
    if (!require_device()) return 0;
    const uint32_t sms = sm_count();
    RC_REQUIRE(sms, "kv attend: the device's size is not known");
    return attend_workspace(sms * kv_blocks(val_size(kv->type), kv->head_dim), kv->head_dim);
}

int redcuda_kv_attend_device(const redcuda_paged_kv *kv, const int32_t *table_dev, uint32_t table_width, uint32_t n_seqs, const int32_t *lens_dev,
                             uint32_t n_q, uint32_t q_type, const void *q_dev, uint64_t q_stride, const void *k_new_dev, const void *v_new_dev,
                             uint64_t new_stride, float scale, void *out_dev, float *lse_dev, void *workspace_dev, uint64_t workspace_bytes, void *stream) {
    uint64_t st[3];
    if (!kv_check(kv, "kv attend", st)) return 0;
    RC_REQUIRE(table_dev && lens_dev && q_dev && out_dev && n_seqs && table_width, "kv attend: null or empty argument");
    RC_REQUIRE((k_new_dev != nullptr) == (v_new_dev != nullptr), "kv attend: a new key without a value, or a value without a key");
    RC_REQUIRE(n_q && n_q <= 65535u && n_q % kv->n_kv == 0u, "kv attend: %u query heads over %u K/V heads", n_q, kv->n_kv);
    RC_REQUIRE(n_seqs < 0x7fffffffu && table_width < 0x7fffffffu, "kv attend: too many sequences or pages");
    RC_REQUIRE((uint64_t)table_width * kv->page_size < (1ull << 32), "kv attend: a page table of more than 2^32 positions");
    RC_REQUIRE(q_type == kv->type || (q_type == VT_F32 && kv->type == VT_F16), "kv attend: queries of type %u over a cache of type %u (F32 over F32 or F16, or the cache's own type)", q_type, kv->type);
    const uint32_t qs = val_size(q_type), hd = kv->head_dim;
    const uint64_t qrow = (uint64_t)n_q * hd, nrow = (uint64_t)kv->n_kv * hd;
    if (!q_stride) q_stride = qrow;
    if (!new_stride) new_stride = nrow;
    RC_REQUIRE(q_stride >= qrow && q_stride * qs % 16u == 0u && q_stride < (1ull << 32) && new_stride >= nrow && new_stride * qs % 16u == 0u && new_stride < (1ull << 32),
               "kv attend: row strides %llu and %llu (multiples of 16 bytes, at least a row)", (unsigned long long)q_stride, (unsigned long long)new_stride);
    RC_REQUIRE(aligned16(q_dev) && aligned16(k_new_dev) && aligned16(v_new_dev) && aligned16(out_dev) && aligned16(workspace_dev), "kv attend: a pointer is not 16-byte aligned");
    const uint64_t out_bytes = (uint64_t)n_seqs * qrow * qs;
    // what the call needs of the workspace, which may begin an arena with other arrays of the call behind it; without a device, which refuses the call anyway, all that is given
    const uint32_t sms = sm_count(), most_blocks = sms * kv_blocks(val_size(kv->type), hd);
    const uint64_t need = attend_workspace(most_blocks, hd), ws_bytes = sms && need < workspace_bytes ? need : workspace_bytes;
    RC_REQUIRE(!overlap(out_dev, out_bytes, q_dev, span_bytes(n_seqs, q_stride, qrow, qs)) && !overlap(out_dev, out_bytes, k_new_dev, span_bytes(n_seqs, new_stride, nrow, qs)) &&
               !overlap(out_dev, out_bytes, v_new_dev, span_bytes(n_seqs, new_stride, nrow, qs)), "kv attend: the output lies inside the inputs");
    RC_REQUIRE(aligned4(table_dev) && aligned4(lens_dev) && aligned4(lse_dev), "kv attend: whole numbers or lse are not 4-byte aligned");
    RC_REQUIRE(!kv_overlap(kv, st, out_dev, out_bytes) && !kv_overlap(kv, st, q_dev, span_bytes(n_seqs, q_stride, qrow, qs)) && !kv_overlap(kv, st, workspace_dev, ws_bytes) &&
               !kv_overlap(kv, st, k_new_dev, span_bytes(n_seqs, new_stride, nrow, qs)) && !kv_overlap(kv, st, v_new_dev, span_bytes(n_seqs, new_stride, nrow, qs)) &&
               !kv_overlap(kv, st, lse_dev, (uint64_t)n_seqs * n_q * 4u), "kv attend: rows, output or workspace lie inside the cache");
    const Span written[3] = {{out_dev, out_bytes}, {lse_dev, (uint64_t)n_seqs * n_q * 4u}, {workspace_dev, ws_bytes}};
    const Span read[5] = {{q_dev, span_bytes(n_seqs, q_stride, qrow, qs)}, {k_new_dev, span_bytes(n_seqs, new_stride, nrow, qs)}, {v_new_dev, span_bytes(n_seqs, new_stride, nrow, qs)},
                          {table_dev, (uint64_t)n_seqs * table_width * 4u}, {lens_dev, (uint64_t)n_seqs * 4u}};
    RC_REQUIRE(!spans_overlap(written, read), "kv attend: output, lse or workspace overlap one another or the inputs");
    RC_REQUIRE(!kv_overlap(kv, st, table_dev, read[3].n) && !kv_overlap(kv, st, lens_dev, read[4].n), "kv attend: the page table or the lengths lie inside the cache");
    RC_REQUIRE(!(scale != scale), "kv attend: scale is not a number");
    if (!require_device()) return 0;
    RC_REQUIRE(sms, "kv attend: the device's size is not known");
    RC_REQUIRE(workspace_dev && workspace_bytes >= need, "kv attend: a workspace of %llu bytes is needed", (unsigned long long)need);
    AttendArgs A{};
    A.k = kv->k; A.v = kv->v; A.page_stride = st[0]; A.token_stride = st[1]; A.head_stride = st[2];
    A.table = table_dev; A.table_width = table_width; A.page_size = kv->page_size; A.n_pages = kv->n_pages;
    A.lens = lens_dev; A.n_seqs = n_seqs; A.n_kv = kv->n_kv; A.n_q = n_q; A.G = n_q / kv->n_kv; A.gsplit = (A.G + 7u) / 8u;
    A.q = q_dev; A.q_stride = q_stride; A.k_new = k_new_dev; A.v_new = v_new_dev; A.new_stride = new_stride;
    A.scale_log2 = (float)((scale == 0.f ? 1.0 / sqrt((double)hd) : (double)scale) * 1.4426950408889634074);
    A.out = out_dev; A.lse = lse_dev; A.status = status_words();
    // no more blocks than there can be runs of tiles
    const uint64_t half = kv_half(val_size(kv->type), hd), tile = half / (hd * val_size(kv->type)), tiles = ((uint64_t)table_width * kv->page_size + tile - 1u) / tile;
    auto few = [](uint64_t n) { return n < 8192u ? n : 8192u; };      // more than that of one thing is blocks enough
    const uint64_t runs = (few(tiles) * few(n_seqs) * few(A.n_kv * A.gsplit) + KV_MIN_TILES - 1u) / KV_MIN_TILES;
    const uint32_t blocks = runs < most_blocks ? (uint32_t)runs : most_blocks;
    // one launch for few heads of moderate length
    const uint64_t heads = (uint64_t)n_seqs * A.n_kv * A.gsplit;
    const uint64_t most_tiles = (uint64_t)KV_CLUSTER * KV_WARPS * (kv->type == VT_F32 ? KV_CLUSTER_TILES_F32 * (8192u / half) : KV_CLUSTER_TILES);
    A.clusters = heads <= KV_CLUSTER_HEADS && heads * KV_CLUSTER <= (uint64_t)sms * KV_BLOCKS && tiles <= most_tiles ? (uint32_t)heads : 0u;
    A.meta = (uint32_t *)workspace_dev;
    A.part = (float *)(A.meta + (size_t)blocks * 4u);
    A.part_ml = A.part + (size_t)blocks * 2u * 8u * hd;
    cudaStream_t s = (cudaStream_t)stream;
    if (kv->type == VT_F32) return launch_attend_hd<float, float>(A, hd, blocks, s);
    if (kv->type == VT_BF16) return launch_attend_hd<__nv_bfloat16, __nv_bfloat16>(A, hd, blocks, s);
    return q_type == VT_F32 ? launch_attend_hd<__half, float>(A, hd, blocks, s) : launch_attend_hd<__half, __half>(A, hd, blocks, s);
}

}  // extern "C"
