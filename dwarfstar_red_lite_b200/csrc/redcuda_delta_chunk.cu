// The gated delta rule of whole prompts in chunks of 64 tokens on the tensor cores (states of 128). With G_t the sum of the chunk's gates up to token t, k_t, q_t, v_t its rows, S the state
// before the chunk (rows: values), the corrections d_t of a chunk solve a triangular system, the rest is products:
//     (1 + A) D = beta R,    A[t][s] = beta_t exp(G_t - G_s) k_t . k_s  (s < t),    R_t = v_t - exp(G_t) S k_t
//     out_t = scale (exp(G_t) S q_t + sum_{s <= t} P[t][s] d_s),   P[t][s] = exp(G_t - G_s) q_t . k_s
//     S    <- exp(G_last) S + sum_s exp(G_last - G_s) d_s k_s^T
// What does not depend on the state, T = (1 + A)^-1 beta and P, is made for all chunks at once by k_delta_prep; k_delta_chunk then takes a state through its sequence's chunks.
//
// Precision: the state and every sum are fp32; operands are fp16 digits under a power of two, two of them (22 bits) where the number is computed or given in fp32, one
// where it is given in 16 bits, and products of lower digits with one another are left out (2^-22 of a product).
// Values that are not finite must not reach a product with a zero of the triangle: they are taken out, and from their token on what depends on them is NaN.
#include "redcuda_delta.cuh"
#include "redcuda_tc_gemm.cuh"

#include <math.h>
#include <type_traits>

namespace rc {

constexpr int DC_T = 64, DC_S = 128;             // tokens of a chunk; the state
// Operand tiles as the MMAs read them (K-major, no swizzle): [k / 8][row][8 values], 16 bytes a row and piece.
constexpr uint32_t DC_KQ = 2u * DC_T * DC_S * 2u;        // a digit of the chunk's keys (rows 0 .. 63) and queries (64 .. 127), k: the state's columns
constexpr uint32_t DC_KT = DC_T * DC_S * 2u;             // a digit of the keys transposed: rows: the state's columns, k: tokens
constexpr uint32_t DC_SQ = DC_T * DC_T * 2u;             // a digit of T or P, rows t, k: s
struct DcMeta {                                  // of a chunk and value head
    float dec[DC_T], kdec[DC_T];                 // exp(G_t), exp(G_last - G_t)
    float last, f_k, f_q, f_t[4], f_p[4];        // exp(G_last); what a digit's unit is worth in K, in Q, in 16 rows each of T and P
    float most_dec, most_kdec, t_sum[4];         // the largest exp(G_t) and exp(G_last - G_t); the largest sum of magnitudes of a row, in 16 rows each of T
    uint32_t nan_from, bad_q[2], pad[108];       // tokens from which on everything is NaN; tokens whose query is not finite
};
static_assert(sizeof(DcMeta) == 1024, "copied in whole");
constexpr uint32_t DC_REC = 4u * DC_SQ + (uint32_t)sizeof(DcMeta);       // T hi, T lo, P hi, P lo, meta
__host__ __device__ constexpr uint32_t dc_keys(int dig) { return (uint32_t)dig * (DC_KQ + DC_KT); }      // KQ hi (, lo), KT hi (, lo)

// A call's chunks are numbered through, sequence by sequence. Bounds that cannot be count no chunk, so that the others' numbers are theirs alone whatever those are. Sequences that have no rows in common
// have n_tokens / 64 + n_seqs chunks at most; one whose chunks lie beyond that (others claim the same rows) is left out.
// Up to DC_NEAR sequences every block counts for itself, a sequence a lane. Of more, k_delta_plan writes to the workspace what a block needs to know (the plan).
constexpr uint32_t DC_NEAR = 32u;
struct alignas(16) DcSeq { uint32_t b, first; int32_t lo, hi; };             // the sequence, the number of its first chunk, its bounds
static uint64_t dc_slots(uint32_t n_tokens, uint32_t n_seqs) { return (uint64_t)n_tokens / DC_T + n_seqs; }
__device__ __forceinline__ uint32_t dc_chunks(int32_t lo, int32_t hi, uint32_t n_tokens) {
    return lo < 0 || hi < lo || (uint32_t)hi > n_tokens ? 0u : ((uint32_t)(hi - lo) + DC_T - 1u) / DC_T;
}
__device__ __forceinline__ uint32_t dc_warp_sum_to(uint32_t x) {             // of the lanes up to this one
    const uint32_t lane = threadIdx.x & 31u;
#pragma unroll
    for (int w = 1; w < 32; w <<= 1) { const uint32_t y = __shfl_up_sync(0xffffffffu, x, w); if (lane >= (uint32_t)w) x += y; }
    return x;
}
// The i-th longest sequence, to shared memory, for the whole block (it meets a barrier). Blocks of long sequences go first.
__device__ __forceinline__ void dc_seq(const DeltaArgs &A, uint32_t n_seqs, const DcSeq *plan, uint32_t i, DcSeq &to) {
    const uint32_t lane = threadIdx.x;
    if (n_seqs > DC_NEAR) {
        if (lane == 0u) *reinterpret_cast<uint4 *>(&to) = *reinterpret_cast<const uint4 *>(plan + i);
    } else if (lane < 32u) {
        int32_t lo = 0, hi = 0;
        if (lane < n_seqs) { lo = A.cu[lane]; hi = A.cu[lane + 1u]; }
        const uint32_t n = dc_chunks(lo, hi, A.n_tokens), first = dc_warp_sum_to(n) - n;
        uint32_t before = 0u;                    // longer ones, and equal ones ahead of it
        for (uint32_t j = 0; j < n_seqs; ++j) { const uint32_t other = __shfl_sync(0xffffffffu, n, (int)j); before += other > n || (other == n && j < lane); }
        if (lane < n_seqs && before == i) to = DcSeq{lane, first, lo, hi};
    }
    __syncthreads();
}
// the plan's second part: the numbers of the sequences' first chunks, in their own order
template <class P> __device__ __forceinline__ auto dc_firsts(P *plan, uint32_t n_seqs) { return reinterpret_cast<typename std::conditional<std::is_const<P>::value, const uint32_t, uint32_t>::type *>(plan + n_seqs); }
// the bounds of the sequence that chunk number `slot` belongs to, and which of its chunks that is, or false: none (for a whole warp)
__device__ __forceinline__ bool dc_find(const DeltaArgs &A, uint32_t n_seqs, const DcSeq *plan, uint32_t slot, int32_t &lo, int32_t &hi, uint32_t &chunk) {
    const uint32_t lane = threadIdx.x & 31u;
    if (n_seqs <= DC_NEAR) {
        lo = hi = 0;
        if (lane < n_seqs) { lo = A.cu[lane]; hi = A.cu[lane + 1u]; }
        const uint32_t n = dc_chunks(lo, hi, A.n_tokens), end = dc_warp_sum_to(n), m = __ballot_sync(0xffffffffu, slot < end);
        if (!m) return false;
        const int b = __ffs((int)m) - 1;
        chunk = slot - __shfl_sync(0xffffffffu, end - n, b);
        lo = __shfl_sync(0xffffffffu, lo, b); hi = __shfl_sync(0xffffffffu, hi, b);
        return true;
    }
    const uint32_t *const firsts = dc_firsts(plan, n_seqs);
    uint32_t cnt = n_seqs, b = 0u;               // the last sequence whose first chunk is no later: one that has chunks, unless slot is behind the last
    while (cnt > 1u) {
        const uint32_t step = (cnt + 31u) / 32u, i = lane * step, m = __ballot_sync(0xffffffffu, i < cnt && firsts[b + i] <= slot), at = (31u - (uint32_t)__clz((int)m)) * step;
        cnt = min(step, cnt - at); b += at;
    }
    chunk = slot - firsts[b];
    lo = A.cu[b]; hi = A.cu[b + 1u];
    return chunk < dc_chunks(lo, hi, A.n_tokens);
}

// One block: the plan of more than DC_NEAR sequences. A thread has a run of them; the order is by number of chunks, those of DC_KINDS and more alike (how they lie among themselves changes no result).
// 1024 sequences of 64 tokens, 32 heads over 16: 3.2 ms in all; with every block of k_delta_chunk finding its sequence's place for itself 19.4, up to 256 sequences 1.07 -> 0.82.
constexpr uint32_t DC_KINDS = 1024u;
__global__ void __launch_bounds__(1024) k_delta_plan(DeltaArgs A, uint32_t n_seqs, DcSeq *plan) {
    pdl_prologue();
    __shared__ uint64_t s_sum[32];
    __shared__ uint32_t s_kind[DC_KINDS], s_part[32];        // sequences with so many chunks; where the next of them goes
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, per = (n_seqs + 1023u) / 1024u, b0 = min(n_seqs, tid * per), b1 = min(n_seqs, b0 + per);
    static_assert(DC_KINDS == 1024u, "one a thread");
    s_kind[tid] = 0u;
    __syncthreads();
    uint64_t mine = 0u;
    for (uint32_t b = b0; b < b1; ++b) {
        const uint32_t n = dc_chunks(A.cu[b], A.cu[b + 1u], A.n_tokens);
        mine += n;
        atomicAdd(&s_kind[min(n, DC_KINDS - 1u)], 1u);
    }
    uint64_t at = mine;
#pragma unroll
    for (int w = 1; w < 32; w <<= 1) { const uint64_t y = __shfl_up_sync(0xffffffffu, at, w); if (lane >= (uint32_t)w) at += y; }
    if (lane == 31u) s_sum[warp] = at;
    __syncthreads();
    for (uint32_t w = 0; w < warp; ++w) at += s_sum[w];
    at -= mine;
    const uint32_t kind = DC_KINDS - 1u - tid, many = s_kind[kind], upto = dc_warp_sum_to(many);       // thread 0 has the longest
    if (lane == 31u) s_part[warp] = upto;
    __syncthreads();
    uint32_t to = upto - many;
    for (uint32_t w = 0; w < warp; ++w) to += s_part[w];
    s_kind[kind] = to;
    __syncthreads();
    for (uint32_t b = b0; b < b1; ++b) {
        const int32_t lo = A.cu[b], hi = A.cu[b + 1u];
        const uint32_t n = dc_chunks(lo, hi, A.n_tokens), first = (uint32_t)min(at, (uint64_t)0xffffffffu);
        at += n;
        dc_firsts(plan, n_seqs)[b] = first;
        plan[atomicAdd(&s_kind[min(n, DC_KINDS - 1u)], 1u)] = DcSeq{b, first, lo, hi};
    }
}

__device__ __forceinline__ uint32_t dc_kq_at(uint32_t row, uint32_t piece) { return piece * 2048u + row * 16u; }       // of KQ, and of KT
__device__ __forceinline__ uint32_t dc_sq_at(uint32_t row, uint32_t piece) { return piece * 1024u + row * 16u; }
__device__ __forceinline__ uint32_t dc_smem(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
// 2^e that brings `most` into [2^14, 2^15) (fp16 holds 2^15.99), and its reciprocal
__device__ __forceinline__ void dc_scale(float most, float &up, float &unit) {
    int e = 0;
    if (most > 0.f && most < INFINITY) e = min(141 - (int)(__float_as_uint(most) >> 23), 126);
    up = __uint_as_float((uint32_t)(127 + e) << 23);
    unit = __uint_as_float((uint32_t)(127 - e) << 23);
}
__device__ __forceinline__ uint32_t dc_pack(float a, float b) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t *>(&h); }
__device__ __forceinline__ void dc_digits(float a, float b, uint32_t &hi, uint32_t &lo) {
    hi = dc_pack(a, b);
    const float2 h = __half22float2(*reinterpret_cast<const __half2 *>(&hi)), l = __fadd2_rn(make_float2(a, b), make_float2(-h.x, -h.y));
    lo = dc_pack(l.x, l.y);
}
__device__ __forceinline__ void dc_ldsm(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void dc_ldsm_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void dc_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// ---- what does not depend on the state ----------------------------------------------------------------------------------------------------------
// A block per chunk and key head: digits of K and Q (a power of two for the chunk's keys, one for its queries), K K^T and Q K^T on the tensor cores (their lower triangles, 16 rows a warp, which stay in its
// registers), then for the key head's value heads, two at a time, the decays, P and its digits from the registers, A to shared memory, the inverse of 1 + A and the digits of T. The inverse goes by blocks
// of 16: those on the diagonal by substitution, a column a lane; the others T_ij = -T_ii sum_k A_ik T_kj, a column of blocks a warp, which is as stable as substitution (powers of A are not, where
// keys are alike). The digits of T and P have a power of two for 16 rows each, so that no warp waits for another's largest.
// What bounds it is latency: a dozen short phases between barriers, hence three blocks an SM. 16 key heads with 2 value heads each: a prompt of 2000 tokens in F32 (512 blocks) 45 us, twelve prompts
// of 16384 tokens together in BF16 (some 4200 blocks) 178 us. One exponent for a chunk's keys and one for its queries: a key 2^17 smaller than the largest still has its 22 bits, a smaller one loses some.
constexpr uint32_t DC_PITCH = 68u;               // floats of a row of the 64 x 64 matrices in shared memory
constexpr uint32_t DC_MAT = DC_T * DC_PITCH * 4u;
__device__ __forceinline__ void dc_half_sync(uint32_t half) { asm volatile("bar.sync %0, 128;" :: "r"(half + 1u) : "memory"); }
__device__ __forceinline__ float dc_warp_max(float x) { return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(x))); }      // of numbers that are not negative
// e^x for x <= 0 (and moderate x above): the error of the argument is |x| 2^-24, of a result e^x
__device__ __forceinline__ float dc_exp(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.44269504088896340736f)); return r; }
// The digits of a 16 x 16 block in the accumulator layout (8 values a lane) as operand A, under the block's own power of two
__device__ __forceinline__ float dc_block_operand(const float (&x)[2][4], uint32_t (&hi)[4], uint32_t (&lo)[4]) {
    float most = 0.f, up, unit;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) most = fmaxf(most, fabsf(x[i][e]));
    dc_scale(dc_warp_max(most), up, unit);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        dc_digits(x[i][0] * up, x[i][1] * up, hi[2 * i], lo[2 * i]);
        dc_digits(x[i][2] * up, x[i][3] * up, hi[2 * i + 1], lo[2 * i + 1]);
    }
    return unit;
}
// c += (hi + lo) * B, B[k][n] = m[n][k] a block of a matrix in shared memory, its digits under `up`
__device__ __forceinline__ void dc_block_product(float (&c)[2][4], const uint32_t (&hi)[4], const uint32_t (&lo)[4], const float *m, float up) {
    const uint32_t g = (threadIdx.x & 31u) >> 2, c2 = (threadIdx.x & 3u) * 2u;
#pragma unroll
    for (int i = 0; i < 2; ++i) {                // n: rows 8 i .. 8 i + 7 of the block
        uint32_t bh[2], bl[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const float2 x = *reinterpret_cast<const float2 *>(m + (i * 8 + g) * DC_PITCH + k * 8 + c2);
            dc_digits(x.x * up, x.y * up, bh[k], bl[k]);
        }
        dc_mma(c[i], lo, bh[0], bh[1]);
        dc_mma(c[i], hi, bl[0], bl[1]);
        dc_mma(c[i], hi, bh[0], bh[1]);
    }
}

// WIDE: more than two value heads a key head (the products are then kept for the next two, which spills 136 to 168 bytes a thread)
template <class T, int DIG, bool WIDE>
__global__ void __launch_bounds__(256, 3) k_delta_prep(DeltaArgs A, uint32_t n_seqs, uint8_t *ws, uint64_t slots, const DcSeq *plan) {
    pdl_prologue();
    extern __shared__ __align__(128) uint8_t sm[];           // the digits; then the matrices A and T of two value heads
    __shared__ float s_red[2][8], s_beta[2][DC_T], s_diag[2][4], s_amax[2][4], s_peak[2];
    __shared__ float2 s_cum[2][DC_T];            // the sums of the gates, each as a float and what it lacks
    __shared__ uint32_t s_bad[2][2];             // tokens whose key or query is not finite
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, kh = blockIdx.y, width = A.rank / A.groups;
    const uint64_t slot = blockIdx.x;
    int32_t lo, hi;
    uint32_t chunk;
    if (!dc_find(A, n_seqs, plan, blockIdx.x, lo, hi, chunk)) return;
    const uint32_t t0 = (uint32_t)lo + chunk * DC_T, n = min((uint32_t)DC_T, (uint32_t)hi - t0);
    uint8_t *const keys = ws + (slot * A.groups + kh) * dc_keys(DIG), *const recs = ws + slots * A.groups * dc_keys(DIG) + slot * A.rank * DC_REC;
    const uint32_t dv = warp == 0u ? 0u : warp == 7u ? 1u : 2u;          // the value head of a pair whose decays this warp makes (2: none): the warps with the fewest products

    float g_raw[2] = {0.f, 0.f}, b_raw[2] = {0.f, 0.f};      // gates and betas of tokens 2 lane and 2 lane + 1
    auto gates = [&](uint32_t v) {
#pragma unroll
        for (uint32_t i = 0; i < 2u; ++i) {
            g_raw[i] = b_raw[i] = 0.f;
            if (lane * 2u + i < n) {
                g_raw[i] = A.gate[(uint64_t)(t0 + lane * 2u + i) * A.rank + kh * width + v];
                b_raw[i] = A.beta[(uint64_t)(t0 + lane * 2u + i) * A.rank + kh * width + v];
            }
        }
    };
    float f_k, f_q;
    {   // rows 8 warp .. 8 warp + 7 of K and Q: a lane has row lane % 8 and the 8-value pieces lane / 8 + 4 i
        constexpr int P = 8 * sizeof(T) / 16, N = 16 / sizeof(T);      // loads of eight values, values of a load
        const uint32_t t = warp * 8u + (lane & 7u);
        uint4 rk[4][P], rq[4][P];
        const T *const k = reinterpret_cast<const T *>(A.k) + (uint64_t)(t0 + min(t, n - 1u)) * A.k_stride + kh * DC_S + (lane >> 3) * 8u;
        const T *const q = reinterpret_cast<const T *>(A.q) + (uint64_t)(t0 + min(t, n - 1u)) * A.q_stride + kh * DC_S + (lane >> 3) * 8u;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < P; ++e) { rk[i][e] = reinterpret_cast<const uint4 *>(k + i * 32)[e]; rq[i][e] = reinterpret_cast<const uint4 *>(q + i * 32)[e]; }
        if (dv < min(width, 2u)) gates(dv);
        if (tid < 4u) s_bad[tid >> 1][tid & 1u] = 0u;
        __syncthreads();
        // a row's largest; a row behind the last token or with a number that is not finite is taken out
        auto values = [](uint4 w, float (&x)[N]) {
            const T *const p = reinterpret_cast<const T *>(&w);
#pragma unroll
            for (int e = 0; e < N; ++e) x[e] = to_f32(p[e]);
        };
        auto most_of = [&](uint4 (&r)[4][P], uint32_t (&bad)[2]) {
            float most = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < P; ++e) {
                    float x[N];
                    values(r[i][e], x);
#pragma unroll
                    for (int j = 0; j < N; ++j) asm("max.NaN.f32 %0, %0, %1;" : "+f"(most) : "f"(fabsf(x[j])));
                }
            const bool out = __ballot_sync(0xffffffffu, !(most < INFINITY)) & (0x01010101u << (lane & 7u));
            if (out && t < n && lane < 8u) atomicOr(&bad[t >> 5], 1u << (t & 31u));
            if (out || t >= n) {
                most = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < P; ++e) r[i][e] = make_uint4(0u, 0u, 0u, 0u);
            }
            return dc_warp_max(most);
        };
        float mk = most_of(rk, s_bad[0]), mq = most_of(rq, s_bad[1]);
        if (lane == 0u) { s_red[0][warp] = mk; s_red[1][warp] = mq; }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) { mk = fmaxf(mk, s_red[0][i]); mq = fmaxf(mq, s_red[1][i]); }
        float up_k, up_q;
        dc_scale(mk, up_k, f_k);
        dc_scale(mq, up_q, f_q);
        auto put = [&](const uint4 (&r)[P], float up, uint32_t at) {
            uint32_t h[4], l[4];
#pragma unroll
            for (int e = 0; e < P; ++e) {
                float x[N];
                values(r[e], x);
#pragma unroll
                for (int j = 0; j < N; j += 2) dc_digits(x[j] * up, x[j + 1] * up, h[(e * N + j) / 2], l[(e * N + j) / 2]);
            }
            *reinterpret_cast<uint4 *>(sm + at) = *reinterpret_cast<const uint4 *>(h);
            *reinterpret_cast<uint4 *>(keys + at) = *reinterpret_cast<const uint4 *>(h);
            if (DIG == 2) { *reinterpret_cast<uint4 *>(sm + DC_KQ + at) = *reinterpret_cast<const uint4 *>(l); *reinterpret_cast<uint4 *>(keys + DC_KQ + at) = *reinterpret_cast<const uint4 *>(l); }
        };
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
            put(rk[i], up_k, dc_kq_at(t, (lane >> 3) + 4u * i));
            put(rq[i], up_q, dc_kq_at(DC_T + t, (lane >> 3) + 4u * i));
        }
        __syncthreads();
    }
    // the keys transposed: 8 x 8 blocks turned by ldmatrix; warp: eight tokens, four blocks of eight columns at a time
#pragma unroll
    for (uint32_t d = 0; d < (uint32_t)DIG; ++d)
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
            uint32_t x[4];
            dc_ldsm_t(x, dc_smem(sm) + d * DC_KQ + dc_kq_at(warp * 8u + (lane & 7u), i * 4u + (lane >> 3)));
#pragma unroll
            for (uint32_t j = 0; j < 4u; ++j)
                *reinterpret_cast<uint32_t *>(keys + DIG * DC_KQ + d * DC_KT + dc_kq_at((i * 4u + j) * 8u + (lane >> 2), warp) + (lane & 3u) * 4u) = x[j];
        }
    // The decays of a value head, by one warp: tokens 2 lane and 2 lane + 1. The sums of the gates are kept as a float and what it lacks: differences of long sums are wanted to 2^-24 of themselves.
    auto decays = [&](uint32_t v) {
        DcMeta *const meta = reinterpret_cast<DcMeta *>(recs + (uint64_t)(kh * width + v) * DC_REC + 4u * DC_SQ);
        auto add = [](float2 x, float2 y) {      // (x.x + x.y) + (y.x + y.y)
            const float s = x.x + y.x, z = s - x.x, e = ((x.x - (s - z)) + (y.x - z)) + (x.y + y.y), r = s + e;
            return make_float2(r, e - (r - s));
        };
        float2 g[2];
        float bt[2];
        bool bad[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t t = lane * 2u + i;
            bad[i] = !(g_raw[i] < INFINITY) || !(fabsf(b_raw[i]) < INFINITY) || ((s_bad[0][t >> 5] >> (t & 31u)) & 1u);
            g[i] = make_float2(bad[i] ? 0.f : g_raw[i] < -200.f ? -200.f : g_raw[i], 0.f);      // exp is 0 from -104 on; -infinity cuts the past off
            bt[i] = bad[i] ? 0.f : b_raw[i];
        }
        g[1] = add(g[0], g[1]);
        float2 sum = g[1];
        for (int w = 1; w < 32; w <<= 1) {
            const float2 x = make_float2(__shfl_up_sync(0xffffffffu, sum.x, w), __shfl_up_sync(0xffffffffu, sum.y, w));
            if (lane >= (uint32_t)w) sum = add(x, sum);
        }
        const float2 last = make_float2(__shfl_sync(0xffffffffu, sum.x, 31), __shfl_sync(0xffffffffu, sum.y, 31));
        float2 before = make_float2(__shfl_up_sync(0xffffffffu, sum.x, 1), __shfl_up_sync(0xffffffffu, sum.y, 1));
        if (lane == 0u) before = make_float2(0.f, 0.f);
        const float2 G[2] = {add(before, g[0]), sum};
        const uint32_t m0 = __ballot_sync(0xffffffffu, bad[0]), m1 = __ballot_sync(0xffffffffu, bad[1]);
        const uint32_t first0 = m0 ? 2u * ((uint32_t)__ffs((int)m0) - 1u) : (uint32_t)DC_T, first1 = m1 ? 2u * ((uint32_t)__ffs((int)m1) - 1u) + 1u : (uint32_t)DC_T;
        float dec[2], kdec[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            dec[i] = expf(G[i].x + G[i].y); kdec[i] = expf((last.x - G[i].x) + (last.y - G[i].y));
            s_cum[v & 1u][lane * 2u + i] = G[i]; s_beta[v & 1u][lane * 2u + i] = bt[i];
        }
        *reinterpret_cast<float2 *>(&meta->dec[lane * 2u]) = make_float2(dec[0], dec[1]);
        *reinterpret_cast<float2 *>(&meta->kdec[lane * 2u]) = make_float2(kdec[0], kdec[1]);
        const float most_dec = dc_warp_max(fmaxf(dec[0], dec[1])), most_kdec = dc_warp_max(fmaxf(kdec[0], kdec[1]));
        // the largest exp(G_t - G_s), s <= t: 1 unless a gate is positive
        float low = fminf(G[0].x, G[1].x);
        for (int w = 1; w < 32; w <<= 1) { const float x = __shfl_up_sync(0xffffffffu, low, w); if (lane >= (uint32_t)w) low = fminf(low, x); }
        float ahead = __shfl_up_sync(0xffffffffu, low, 1);
        if (lane == 0u) ahead = INFINITY;
        const float rise = fmaxf(fmaxf(G[0].x - fminf(ahead, G[0].x), G[1].x - low), 0.f), peak = expf(dc_warp_max(rise));
        if (lane == 0u) {
            s_peak[v & 1u] = peak;
            meta->last = expf(last.x + last.y); meta->f_k = f_k; meta->f_q = f_q; meta->most_dec = most_dec; meta->most_kdec = most_kdec;
            meta->nan_from = min(first0, first1); meta->bad_q[0] = s_bad[1][0]; meta->bad_q[1] = s_bad[1][1];
        }
    };
    if (dv < min(width, 2u)) decays(dv);
    // warps 0-3: K K^T, rows 16 warp on; 4-7: Q K^T, rows 16 (7 - warp) on, so that every scheduler has as much; the columns up to the diagonal
    const uint32_t which = warp >> 2, mt = which ? 7u - warp : warp, g = lane >> 2, c2 = (lane & 3u) * 2u;
    float c[4][2][4];
    {
        const uint32_t at = dc_smem(sm), ar = which * DC_T + mt * 16u + (lane & 15u), ac = lane >> 4, br = (lane & 7u) + (lane >> 4) * 8u, bc = (lane >> 3) & 1u;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) c[i][j][e] = 0.f;
#pragma unroll 2
        for (uint32_t s = 0; s < 8u; ++s) {
            uint32_t ah[4], al[4];
            dc_ldsm(ah, at + dc_kq_at(ar, 2u * s + ac));
            if (DIG == 2) dc_ldsm(al, at + DC_KQ + dc_kq_at(ar, 2u * s + ac));
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i)
                if (i <= mt) {
                    uint32_t x[4];
                    dc_ldsm(x, at + dc_kq_at(i * 16u + br, 2u * s + bc));
                    dc_mma(c[i][0], ah, x[0], x[1]); dc_mma(c[i][1], ah, x[2], x[3]);
                    if (DIG == 2) {
                        dc_mma(c[i][0], al, x[0], x[1]); dc_mma(c[i][1], al, x[2], x[3]);
                        dc_ldsm(x, at + DC_KQ + dc_kq_at(i * 16u + br, 2u * s + bc));
                        dc_mma(c[i][0], ah, x[0], x[1]); dc_mma(c[i][1], ah, x[2], x[3]);
                    }
                }
        }
        const float f = (which ? f_q : f_k) * f_k;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) c[i][j][e] *= f;
    }
    const uint32_t half = warp >> 2, hw = half ? 3u - (warp & 3u) : warp;         // for the inverse, half a block has a value head; the first block columns have the most to do, so the second half counts backwards: a scheduler has warps w and w + 4
    float *const s_a = reinterpret_cast<float *>(sm + half * 2u * DC_MAT), *const s_t = s_a + DC_T * DC_PITCH;
    float most_c = 0.f;                          // of the warp's products
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) most_c = fmaxf(most_c, fabsf(c[i][j][e]));
    most_c = dc_warp_max(most_c);
    uint32_t v0 = 0u;
    do {
        if (WIDE && v0) {
            __syncthreads();                     // the matrices and decays of the last two have been read
            if (v0 + dv < width && dv < 2u) { gates(v0 + dv); decays(v0 + dv); }
        }
        __syncthreads();                         // the digits have been read; the decays are there
#pragma unroll 1
        for (uint32_t v = v0; v < v0 + 2u && v < width; ++v) {
            const uint32_t o = v & 1u, t = mt * 16u + g;     // rows t and t + 8
            const float2 G0 = s_cum[o][t], G1 = s_cum[o][t + 8u];
            const float b0 = which ? 1.f : s_beta[o][t], b1 = which ? 1.f : s_beta[o][t + 8u];
            uint8_t *const rec = recs + (uint64_t)(kh * width + v) * DC_REC;
            float *const s_to = reinterpret_cast<float *>(sm + o * 2u * DC_MAT) + t * DC_PITCH + c2;
            float up, unit, most = 0.f;
            dc_scale(fminf(most_c * s_peak[o], 3e38f), up, unit);        // of P, from its bound
            if (which && lane == 0u) reinterpret_cast<DcMeta *>(rec + 4u * DC_SQ)->f_p[mt] = unit;
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i)
                if (i <= mt)
#pragma unroll
                    for (uint32_t j = 0; j < 2u; ++j) {
                        float y[4];
#pragma unroll
                        for (uint32_t e = 0; e < 2u; ++e) {
                            const uint32_t s = i * 16u + j * 8u + c2 + e;
                            const float2 Gs = s_cum[o][s];
                            const float x0 = b0 * c[i][j][e] * dc_exp((G0.x - Gs.x) + (G0.y - Gs.y)), x1 = b1 * c[i][j][e + 2] * dc_exp((G1.x - Gs.x) + (G1.y - Gs.y));
                            y[e] = s < t + which ? x0 : 0.f;             // s < t for A, s <= t for P
                            y[e + 2] = s < t + 8u + which ? x1 : 0.f;
                        }
                        if (which) {             // P
#pragma unroll
                            for (uint32_t r = 0; r < 2u; ++r) {
                                uint32_t h, l;
                                dc_digits(y[2u * r] * up, y[2u * r + 1u] * up, h, l);
                                uint8_t *const to = rec + 2u * DC_SQ + dc_sq_at(t + 8u * r, i * 2u + j) + c2 * 2u;
                                *reinterpret_cast<uint32_t *>(to) = h;
                                *reinterpret_cast<uint32_t *>(to + DC_SQ) = l;
                            }
                        } else {
                            *reinterpret_cast<float2 *>(s_to + i * 16u + j * 8u) = make_float2(y[0], y[1]);
                            *reinterpret_cast<float2 *>(s_to + 8u * DC_PITCH + i * 16u + j * 8u) = make_float2(y[2], y[3]);
                            most = fmaxf(fmaxf(fmaxf(most, fabsf(y[0])), fmaxf(fabsf(y[1]), fabsf(y[2]))), fabsf(y[3]));
                        }
                    }
            most = dc_warp_max(most);
            if (!which && lane == 0u) s_amax[o][mt] = most;
        }
        __syncthreads();
        if (v0 + half >= width) { v0 += 2u; continue; }
        uint8_t *const rec = recs + (uint64_t)(kh * width + v0 + half) * DC_REC;
        // the diagonal blocks of the inverse: warp hw has block hw, lane c column c
        {
            const uint32_t o = hw * 16u, col = lane & 15u;
            float x[16], most_t = 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                float e = (uint32_t)r == col ? 1.f : 0.f;
#pragma unroll
                for (int k = 0; k < r; ++k) e = fmaf(-s_a[(o + r) * DC_PITCH + o + k], x[k], e);
                x[r] = e;
                most_t = fmaxf(most_t, fabsf(e));
            }
            if (lane < 16u)
#pragma unroll
                for (int r = 0; r < 16; ++r) s_t[(o + r) * DC_PITCH + o + col] = x[r];
            most_t = dc_warp_max(most_t);
            if (lane == 0u) s_diag[half][hw] = most_t;
        }
        dc_half_sync(half);
        // The others, a column of blocks a warp: X_i = T_ij^T = -(sum_{k < i} X_k A_ik^T) T_ii^T. Transposed, an accumulator is the next product's operand A and rows of A and T_ii are operand B.
        {
            float up_t, unit_t, up_a, unit_a;
            dc_scale(fmaxf(fmaxf(s_diag[half][0], s_diag[half][1]), fmaxf(s_diag[half][2], s_diag[half][3])), up_t, unit_t);
            dc_scale(fmaxf(fmaxf(s_amax[half][0], s_amax[half][1]), fmaxf(s_amax[half][2], s_amax[half][3])), up_a, unit_a);
            const uint32_t j = hw;
            uint32_t xh[3][4], xl[3][4];
            float f[3], x[2][4];
#pragma unroll
            for (int i = 0; i < 2; ++i)          // X_j = T_jj^T
#pragma unroll
                for (int e = 0; e < 4; ++e) x[i][e] = s_t[(j * 16u + i * 8u + c2 + (e & 1)) * DC_PITCH + j * 16u + g + (e >> 1) * 8u];
#pragma unroll
            for (uint32_t d = 0; d < 3u; ++d) {  // block row i = j + d + 1
                const uint32_t i = j + d + 1u;
                if (i >= 4u) break;
                f[d] = dc_block_operand(x, xh[d], xl[d]);
                float m[2][4];
#pragma unroll
                for (int a = 0; a < 2; ++a)
#pragma unroll
                    for (int e = 0; e < 4; ++e) m[a][e] = 0.f;
#pragma unroll
                for (uint32_t k = 0; k <= d; ++k) {
                    float y[2][4];
#pragma unroll
                    for (int a = 0; a < 2; ++a)
#pragma unroll
                        for (int e = 0; e < 4; ++e) y[a][e] = 0.f;
                    dc_block_product(y, xh[k], xl[k], s_a + i * 16u * DC_PITCH + (j + k) * 16u, up_a);
#pragma unroll
                    for (int a = 0; a < 2; ++a)
#pragma unroll
                        for (int e = 0; e < 4; ++e) m[a][e] = fmaf(y[a][e], f[k] * unit_a, m[a][e]);
                }
                uint32_t mh[4], ml[4];
                const float fm = -dc_block_operand(m, mh, ml) * unit_t;
#pragma unroll
                for (int a = 0; a < 2; ++a)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[a][e] = 0.f;
                dc_block_product(x, mh, ml, s_t + i * 16u * DC_PITCH + i * 16u, up_t);
#pragma unroll
                for (int a = 0; a < 2; ++a)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[a][e] *= fm;
                        s_t[(i * 16u + a * 8u + c2 + (e & 1)) * DC_PITCH + j * 16u + g + (e >> 1) * 8u] = x[a][e];
                    }
            }
        }
        dc_half_sync(half);
        // T with its columns' betas: warp hw has 16 rows, a lane every other piece of eight columns of one
        {
            const uint32_t t = hw * 16u + (lane & 15u), p0 = lane >> 4;
            float y[4][8], most = 0.f, sum = 0.f, up, unit;
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i)
                if (i <= hw)
#pragma unroll
                    for (uint32_t e = 0; e < 8u; e += 4u) {
                        const uint32_t s = (p0 + 2u * i) * 8u + e;
                        const float4 x = *reinterpret_cast<const float4 *>(s_t + t * DC_PITCH + s), bt = *reinterpret_cast<const float4 *>(&s_beta[half][s]);
                        y[i][e] = s <= t ? x.x * bt.x : 0.f; y[i][e + 1] = s + 1u <= t ? x.y * bt.y : 0.f;
                        y[i][e + 2] = s + 2u <= t ? x.z * bt.z : 0.f; y[i][e + 3] = s + 3u <= t ? x.w * bt.w : 0.f;
#pragma unroll
                        for (uint32_t a = 0; a < 4u; ++a) { most = fmaxf(most, fabsf(y[i][e + a])); sum += fabsf(y[i][e + a]); }
                    }
            dc_scale(dc_warp_max(most), up, unit);
            sum = dc_warp_max(sum + __shfl_xor_sync(0xffffffffu, sum, 16));
            if (lane == 0u) { reinterpret_cast<DcMeta *>(rec + 4u * DC_SQ)->f_t[hw] = unit; reinterpret_cast<DcMeta *>(rec + 4u * DC_SQ)->t_sum[hw] = sum; }
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i)
                if (i <= hw) {
                    uint4 h, l;
                    dc_digits(y[i][0] * up, y[i][1] * up, h.x, l.x); dc_digits(y[i][2] * up, y[i][3] * up, h.y, l.y);
                    dc_digits(y[i][4] * up, y[i][5] * up, h.z, l.z); dc_digits(y[i][6] * up, y[i][7] * up, h.w, l.w);
                    *reinterpret_cast<uint4 *>(rec + dc_sq_at(t, p0 + 2u * i)) = h;
                    *reinterpret_cast<uint4 *>(rec + DC_SQ + dc_sq_at(t, p0 + 2u * i)) = l;
                }
        }
        v0 += 2u;
    } while (WIDE && v0 < width);
}

// ---- the states through their chunks -------------------------------------------------------------------------------------------------------------
// A block has the 128 rows of one state: row j is lane j of tensor memory, and two threads (of warps w and w + 4) have it in registers, 64 columns each. A chunk is four products on tcgen05,
// with an operand A that the threads write to tensor memory as digits (each row under a scale of its own) and an operand B that bulk copies bring to shared memory:
//     M1  [S k | S q] = S [K | Q]^T      M2  D = R T^T      M4  D' K (the state's)      M3  D P^T (the outputs')
// between them the threads make R of M1's result, D and D' = D exp(G_last - G) of M2's, the new S of M4's, the outputs of M1's and M3's. Of four further warps one issues the products and fetches their
// operands (a tile again as soon as the product that reads it is done), one fetches the values, two store the outputs. What bounds it is the chain M1, R, M2, D', M4, S: each link waits for the one before, so what is
// not a link (the outputs, the digits of D, the largest of S) comes behind the hand-over of one, and M4, S and M1 go by halves of the state's columns, one of the row's two threads behind the other
// (a prompt of 2000 tokens 182 -> 177 us with the preparation, twelve prompts 434 -> 424; M1's keys ahead of its queries 195 and 434: products of 64 columns take as long as those of 128). The scales of R and S come from bounds, which need no exchange between a row's two threads: up to 2^13
// too large costs nothing, as two fp16 digits reach from 2^16 down to 2^-24.
// A chunk takes some 4 us: a prompt of 2000 tokens 127 us (32 blocks), twelve prompts of 16384 tokens together 237 (384 blocks on 148 SMs; tensor cores 26 to 36 % busy).
// The adder of the tensor cores truncates, so lower digits go first and M1's sums are kept in two halves of 64 columns each, which are added in fp32.
constexpr uint32_t DC_THREADS = 384u, DC_ROW_WARPS = 8u, DC_CONTROL = 8u, DC_LOADER = 9u, DC_STORER = 10u;        // 10 and 11 store
// registers: 384 threads are launched with 168 each, of which the four further warps keep 72 and the threads of the rows have 216 (256 x 216 + 128 x 72 = 384 x 168)
constexpr uint32_t DC_REGS_ROWS = 216u, DC_REGS_CONTROL = 72u;
static_assert(256u * DC_REGS_ROWS + 128u * DC_REGS_CONTROL <= 384u * 168u, "a split above the launch's registers waits forever");
enum : uint32_t { DT_S = 0, DT_M1 = 128, DT_D = 128, DT_DK = 192, DT_M4 = 256, DT_R = 384, DT_M3 = 384, DT_M2 = 448 };      // columns of tensor memory; M1: two accumulators of 128
enum : uint32_t { DB_KQ, DB_T, DB_PK, DB_META0, DB_META1, DB_V, DB_M1, DB_M2, DB_M3, DB_M4, DB_M4B, DB_OFREE, DB_R, DB_DK, DB_D, DB_VFREE, DB_OUT, DB_END, DB_S, DB_SB, DB_PAIR, DB_COUNT = DB_PAIR + 4 };
constexpr uint32_t DC_SROW = DC_S * 4u + 16u;    // a row of the state on its way through shared memory, 16 bytes further apart than it is long: a quarter warp's rows lie in different banks
constexpr uint32_t dc_smem_bytes(int dig, uint32_t size) { return dc_keys(dig) + 4u * DC_SQ + 2u * (uint32_t)sizeof(DcMeta) + 2u * DC_T * DC_S * size; }
static_assert(dc_smem_bytes(1, 2u) >= 114u * 1024u && dc_smem_bytes(2, 4u) < 220u * 1024u, "one block an SM: it takes all of the tensor memory");
static_assert(dc_smem_bytes(1, 2u) - DC_KQ >= DC_S * DC_SROW && dc_keys(1) + 4u * DC_SQ >= DC_S * DC_SROW, "the state comes in behind KQ and leaves over the operands");

__device__ __forceinline__ void dc_mma_ts(uint32_t leader, uint32_t d_tmem, uint32_t a_tmem, uint32_t b_desc, uint32_t b_high, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 d;\n\tmov.b64 d, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], d, %4, p;\n\t}\n"
        :: "r"(d_tmem), "r"(a_tmem), "r"(b_desc), "r"(b_high), "r"(idesc), "r"(accumulate), "r"(leader) : "memory");
}
__device__ __forceinline__ void dc_ld16(uint32_t (&r)[16], uint32_t at) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
                   "=r"(r[14]), "=r"(r[15]) : "r"(at));
}
__device__ __forceinline__ void dc_st16(uint32_t at, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
                 :: "r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
                    "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void dc_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// what a warp has stored to tensor memory (and read from it) is done with
__device__ __forceinline__ void dc_hand_over(uint32_t mbar) {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncwarp();
    if ((threadIdx.x & 31u) == 0u) tc_arrive(mbar);
}
// 32 values x f as digits, upper ones to the columns from hi on, lower ones from lo on
__device__ __forceinline__ void dc_put32(const float *x, float f, uint32_t hi, uint32_t lo) {
    uint32_t h[16], l[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float2 y = __fmul2_rn(make_float2(x[2 * i], x[2 * i + 1]), make_float2(f, f));
        dc_digits(y.x, y.y, h[i], l[i]);
    }
    dc_st16(hi, h);
    dc_st16(lo, l);
}

template <class T, int DIG>
__global__ void __launch_bounds__(DC_THREADS, 1) k_delta_chunk(DeltaArgs A, uint32_t n_seqs, const uint8_t *ws, uint64_t slots, const DcSeq *plan) {
    pdl_prologue();
    constexpr uint32_t KEYS = dc_keys(DIG), VROW = DC_S * sizeof(T);
    extern __shared__ __align__(128) uint8_t sm[];
    __shared__ __align__(8) uint64_t s_bar[DB_COUNT];
    __shared__ float s_ex[4][2][DC_S];
    __shared__ uint32_t s_from[2][DC_S], tmem_slot;
    __shared__ volatile uint32_t fail;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const uint32_t h = blockIdx.x, kh = h / (A.rank / A.groups);
    __shared__ DcSeq seq;
    dc_seq(A, n_seqs, plan, A.first_seq + blockIdx.y, seq);
    const int32_t &lo = seq.lo, &hi = seq.hi;     // read where they are wanted: the warps of the rows have no registers for them
    if (lo < 0 || hi < lo || (uint32_t)hi > A.n_tokens) { if (A.status && tid == 0u) A.status[ST_SEQ_BOUNDS] = 1u; return; }
    const int32_t state_slot = delta_slot(A.slots, A.n_slots, seq.b, A.status);
    if (state_slot < 0 || lo == hi) return;
    const uint32_t chunks = ((uint32_t)(hi - lo) + DC_T - 1u) / DC_T;
    if (seq.first + (uint64_t)chunks > slots) { if (A.status && tid == 0u) A.status[ST_SEQ_BOUNDS] = 1u; return; }
    uint8_t *const s_kq = sm, *const s_kt = sm + DIG * DC_KQ, *const s_tt = sm + KEYS, *const s_pp = s_tt + 2u * DC_SQ, *const s_meta = s_tt + 4u * DC_SQ;
    T *const s_v = reinterpret_cast<T *>(s_meta + 2u * sizeof(DcMeta)), *const s_out = s_v + DC_T * DC_S;          // [token][row]
    auto bar = [&](uint32_t i) { return dc_smem(&s_bar[i]); };
    if (tid == 0u) {
        fail = 0u;
        for (uint32_t i = 0; i < DB_COUNT; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(bar(i)), "r"(i >= DB_PAIR || i == DB_OFREE ? 2u : i >= DB_S ? DC_ROW_WARPS / 2u : i >= DB_R ? DC_ROW_WARPS : i == DB_V ? 32u : 1u));
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == DC_CONTROL) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(dc_smem(&tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0), fail_at = dc_smem(const_cast<uint32_t *>(&fail));
    auto wait = [&](uint32_t i, uint32_t parity) { return tc_wait(bar(i), parity & 1u, fail_at); };
    auto expect = [&](uint32_t i, uint32_t bytes) { asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" :: "r"(bar(i)), "r"(bytes) : "memory"); };
    auto copy = [&](uint32_t i, const void *dst, const void *src, uint32_t bytes) {
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" :: "r"(dc_smem(dst)), "l"(src), "r"(bytes), "r"(bar(i)) : "memory");
    };

    if (warp >= DC_CONTROL) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(DC_REGS_CONTROL));
        if (warp == DC_CONTROL) {
            const uint32_t leader = tc_elect();
            const uint64_t slot0 = seq.first;
            const uint8_t *key = ws + (slot0 * A.groups + kh) * KEYS, *rec = ws + slots * A.groups * KEYS + (slot0 * A.rank + h) * DC_REC;      // the next chunk's, as each is asked for
            const uint64_t key_step = (uint64_t)A.groups * KEYS, rec_step = (uint64_t)A.rank * DC_REC;
            auto get_kq = [&](uint32_t c) { if (lane == 0u) { expect(DB_KQ, DIG * DC_KQ); copy(DB_KQ, s_kq, key + c * key_step, DIG * DC_KQ); } };
            auto get_t = [&](uint32_t c) { if (lane == 0u) { expect(DB_T, 2u * DC_SQ); copy(DB_T, s_tt, rec + c * rec_step, 2u * DC_SQ); } };
            auto get_pk = [&](uint32_t c) {
                if (lane == 0u) { expect(DB_PK, 2u * DC_SQ + DIG * DC_KT); copy(DB_PK, s_pp, rec + c * rec_step + 2u * DC_SQ, 2u * DC_SQ); copy(DB_PK, s_kt, key + c * key_step + DIG * DC_KQ, DIG * DC_KT); }
            };
            auto get_meta = [&](uint32_t c) {
                if (lane == 0u) { expect(DB_META0 + (c & 1u), sizeof(DcMeta)); copy(DB_META0 + (c & 1u), s_meta + (c & 1u) * sizeof(DcMeta), rec + c * rec_step + 4u * DC_SQ, sizeof(DcMeta)); }
            };
            get_kq(0u);
            if (wait(DB_S, 0u) && wait(DB_SB, 0u)) { get_meta(0u); get_t(0u); get_pk(0u); }         // over the state, which has been read
            const uint64_t desc = tc_smem_desc(0u, 2048u, 128u), desc_sq = tc_smem_desc(0u, 1024u, 128u);
            const uint32_t high = (uint32_t)(desc >> 32), wide = (uint32_t)desc, slim = (uint32_t)desc_sq;       // the upper words are alike
            const uint32_t b_kq = wide | (dc_smem(s_kq) >> 4), b_kt = wide | (dc_smem(s_kt) >> 4), b_t = slim | (dc_smem(s_tt) >> 4), b_p = slim | (dc_smem(s_pp) >> 4);
            // n columns of results += A B^T over 64 of k, lower digits first. a_lo: columns from A's upper to its lower digits, b_lo: 16-byte units from B's
            auto square = [&](uint32_t n, uint32_t d, uint32_t a, uint32_t a_lo, uint32_t bd, uint32_t b_lo) {
#pragma unroll
                for (uint32_t k = 0; k < 4u; ++k) dc_mma_ts(leader, tmem + d, tmem + a + a_lo + 8u * k, bd + k * 256u, high, tc_idesc(n), k ? 1u : 0u);
                if (DIG == 2)
#pragma unroll
                    for (uint32_t k = 0; k < 4u; ++k) dc_mma_ts(leader, tmem + d, tmem + a + 8u * k, bd + b_lo + k * 256u, high, tc_idesc(n), 1u);
#pragma unroll
                for (uint32_t k = 0; k < 4u; ++k) dc_mma_ts(leader, tmem + d, tmem + a + 8u * k, bd + k * 256u, high, tc_idesc(n), 1u);
            };
            // the same with a lower triangle of 64: a step of 16 of k meets the rows from its own on
            auto triangle = [&](uint32_t d, uint32_t a, uint32_t bd) {
#pragma unroll
                for (uint32_t pass = 0; pass < 3u; ++pass)
#pragma unroll
                    for (uint32_t k = 0; k < 4u; ++k)
                        dc_mma_ts(leader, tmem + d + 16u * k, tmem + a + (pass == 0u ? 32u : 0u) + 8u * k, bd + (pass == 1u ? DC_SQ >> 4 : 0u) + k * (128u + 16u), high, tc_idesc(64u - 16u * k), pass | k ? 1u : 0u);
            };
            uint32_t c = 0u;
#pragma unroll 1
            for (; c < chunks; ++c) {
                const bool more = c + 1u < chunks;
                if (!wait(DB_KQ, c) || (c && !wait(DB_M3, c - 1u)) || !wait(DB_S, c)) break;         // what comes last goes last: a wait takes its time also for what is there
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                square(128u, DT_M1, DT_S, 64u, b_kq, DC_KQ >> 4);
                if (!wait(DB_SB, c)) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                square(128u, DT_M1 + 128u, DT_S + 32u, 64u, b_kq + 4u * 256u, DC_KQ >> 4);
                tc_commit_if(leader, bar(DB_M1));
                if (c) get_pk(c);
                if (!wait(DB_M1, c)) break;
                if (more) get_kq(c + 1u);
                if (!wait(DB_T, c) || !wait(DB_R, c)) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                triangle(DT_M2, DT_R, b_t);
                tc_commit_if(leader, bar(DB_M2));
                if (more) get_meta(c + 1u);
                if (!wait(DB_M2, c)) break;
                if (more) get_t(c + 1u);
                if (!wait(DB_PK, c) || !wait(DB_DK, c)) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                square(64u, DT_M4, DT_DK, 32u, b_kt, DC_KT >> 4);
                tc_commit_if(leader, bar(DB_M4));
                square(64u, DT_M4 + 64u, DT_DK, 32u, b_kt + 64u, DC_KT >> 4);
                tc_commit_if(leader, bar(DB_M4B));
                if (!wait(DB_D, c)) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                triangle(DT_M3, DT_D, b_p);
                tc_commit_if(leader, bar(DB_M3));
            }
            if (!fail) wait(DB_M3, chunks - 1u);
            // where a wait was given up, copies that nobody waits for may still be writing into this block's shared memory: every stage is waited for in both its phases
            if (fail && lane == 0u) for (uint32_t i = DB_KQ; i <= DB_META1; ++i) { mbar_wait(bar(i), 0u); mbar_wait(bar(i), 1u); }
        } else if (warp == DC_LOADER) {          // a chunk's values, 16 bytes a lane and copy (bulk copies of a row each take some hundred cycles apiece)
            constexpr uint32_t PIECES = VROW / 16u;
            const T *const v = reinterpret_cast<const T *>(A.v) + (uint64_t)(uint32_t)lo * A.v_stride + (uint64_t)h * DC_S;
#pragma unroll 1
            for (uint32_t c = 0; c < chunks; ++c) {
                const uint32_t n = min((uint32_t)DC_T, (uint32_t)(hi - lo) - c * DC_T) * PIECES;
                if (c ? !wait(DB_VFREE, c - 1u) : !(wait(DB_S, 0u) && wait(DB_SB, 0u))) break;      // ahead of the first chunk the state is there
#pragma unroll 4
                for (uint32_t i = lane; i < n; i += 32u)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(dc_smem(s_v) + i * 16u), "l"(v + (uint64_t)(c * DC_T + i / PIECES) * A.v_stride + i % PIECES * (16u / sizeof(T))) : "memory");
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" :: "r"(bar(DB_V)) : "memory");
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
        } else {                                 // the outputs, every other row a warp
            constexpr uint32_t PIECES = VROW / 16u;
            const uint32_t first = (warp - DC_STORER) * 32u + lane;
            T *const out = reinterpret_cast<T *>(A.out) + ((uint64_t)(uint32_t)lo * A.rank + h) * DC_S;
#pragma unroll 1
            for (uint32_t c = 0; c < chunks; ++c) {
                const uint32_t n = min((uint32_t)DC_T, (uint32_t)(hi - lo) - c * DC_T) * PIECES;
                if (!wait(DB_OUT, c)) break;
#pragma unroll 4
                for (uint32_t i = first; i < n; i += 64u)
                    *reinterpret_cast<uint4 *>(out + (uint64_t)(c * DC_T + i / PIECES) * A.rank * DC_S + i % PIECES * (16u / sizeof(T))) = *reinterpret_cast<const uint4 *>(s_out + i * (16u / sizeof(T)));
                __syncwarp();
                if (lane == 0u) tc_arrive(bar(DB_OFREE));
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(DC_REGS_ROWS));
        const uint32_t w = warp & 3u, hf = warp >> 2, j = w * 32u + lane, mine = tmem + ((w * 32u) << 16);
        bool ok = true;
        uint32_t met = 0u;
        auto both = [&](float x, uint32_t i) {   // the larger of the row's two; the two warps meet on an mbarrier, whose wait is bounded like the others
            s_ex[i][hf][j] = x;
            __syncwarp();
            if (lane == 0u) tc_arrive(bar(DB_PAIR + w));
            ok &= wait(DB_PAIR + w, met++);
            return fmaxf(x, s_ex[i][hf ^ 1u][j]);
        };
        auto load32 = [&](float (&x)[32], uint32_t col) {
            uint32_t y[2][16];
            dc_ld16(y[0], mine + col);
            dc_ld16(y[1], mine + col + 16u);
            dc_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) x[i] = __uint_as_float(y[i >> 4][i & 15]);
        };
        float *const state = A.state + ((uint64_t)(uint32_t)state_slot * A.rank + h) * DC_S * DC_S;
        float s[64], most_s = 0.f, up, unit_s;
        uint32_t nan = 0u;                       // the row is no number any more
        auto put_s = [&](float bound) {
            dc_scale(bound, up, unit_s);
            dc_put32(s, up, mine + DT_S + hf * 32u, mine + DT_S + 64u + hf * 32u);
            dc_put32(s + 32, up, mine + DT_S + hf * 32u + 16u, mine + DT_S + 64u + hf * 32u + 16u);
            dc_hand_over(bar(DB_S + hf));
        };
        // a warp reads a row at a time and has it from shared memory a row a lane
#pragma unroll
        for (int i = 0; i < 16; ++i) *reinterpret_cast<float4 *>(&s[4 * i]) = *reinterpret_cast<const float4 *>(state + (i * 8u + warp) * DC_S + lane * 4u);
#pragma unroll
        for (int i = 0; i < 16; ++i) *reinterpret_cast<float4 *>(s_kt + (i * 8u + warp) * DC_SROW + lane * 16u) = *reinterpret_cast<const float4 *>(&s[4 * i]);
        asm volatile("bar.sync 1, 256;" ::: "memory");         // all eight warps of the rows come here
#pragma unroll
        for (int i = 0; i < 16; ++i) *reinterpret_cast<float4 *>(&s[4 * i]) = *reinterpret_cast<const float4 *>(s_kt + j * DC_SROW + hf * 256u + i * 16u);
#pragma unroll
        for (int i = 0; i < 64; ++i) { nan |= !(fabsf(s[i]) < INFINITY); most_s = fmaxf(most_s, fabsf(s[i])); }
        s_from[hf][j] = nan;
        most_s = both(most_s, 0u);
        nan |= s_from[hf ^ 1u][j];
        if (nan) {
            most_s = 0.f;
#pragma unroll
            for (int i = 0; i < 64; ++i) s[i] = 0.f;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");           // copies into where the state was come behind its reading
        put_s(most_s);
#pragma unroll 1
        for (uint32_t c = 0; ok && c < chunks; ++c) {
            const DcMeta &M = *reinterpret_cast<const DcMeta *>(s_meta + (c & 1u) * sizeof(DcMeta));
            float r[32], o[32], x[32], unit, most_v = 0.f;
            // the chunk's values, and what they say of R's scale and of the first token from which the row is no number (64: none)
            if (!(ok = wait(DB_META0 + (c & 1u), c >> 1) && wait(DB_V, c))) break;
            uint32_t from = nan ? 0u : M.nan_from;
            {
                const uint32_t n = min((uint32_t)DC_T, (uint32_t)(hi - lo) - c * DC_T);
#pragma unroll
                for (uint32_t i = 0; i < 32u; ++i) r[i] = to_f32(s_v[(hf * 32u + i) * DC_S + j]);
                __syncwarp();
                if (lane == 0u) tc_arrive(bar(DB_VFREE));
                if (n < (uint32_t)DC_T)
#pragma unroll
                    for (uint32_t i = 0; i < 32u; ++i) if (hf * 32u + i >= n) r[i] = 0.f;
#pragma unroll
                for (uint32_t i = 0; i < 32u; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(most_v) : "f"(fabsf(r[i])));
                if (!(most_v < INFINITY)) {
                    most_v = 0.f;
#pragma unroll
                    for (uint32_t i = 0; i < 32u; ++i) {
                        if (!(fabsf(r[i]) < INFINITY)) { from = min(from, hf * 32u + i); r[i] = 0.f; }
                        most_v = fmaxf(most_v, fabsf(r[i]));
                    }
                }
            }
            s_from[hf][j] = from;
            s_ex[2][hf][j] = most_s;
            most_v = both(most_v, 1u);
            if (!ok) break;
            most_s = fmaxf(most_s, s_ex[2][hf ^ 1u][j]);
            from = min(from, s_from[hf ^ 1u][j]);
            const float most_k = 32768.f * M.f_k;        // no key is larger
            dc_scale(fminf(most_v + M.most_dec * (128.f * most_s) * most_k, 3e38f), up, unit);
            if (!(ok = wait(DB_M1, c))) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            {
                load32(o, DT_M1 + hf * 32u);
                load32(x, DT_M1 + 128u + hf * 32u);
                const float f = -unit_s * M.f_k;
#pragma unroll
                for (uint32_t i = 0; i < 32u; ++i) r[i] = fmaf(M.dec[hf * 32u + i] * f, o[i] + x[i], r[i]);
            }
            dc_put32(r, up, mine + DT_R + hf * 16u, mine + DT_R + 32u + hf * 16u);
            dc_hand_over(bar(DB_R));
            {   // the state's part of the outputs
                load32(o, DT_M1 + 64u + hf * 32u);
                load32(x, DT_M1 + 192u + hf * 32u);
                const float f = unit_s * M.f_q;
#pragma unroll
                for (uint32_t i = 0; i < 32u; ++i) o[i] = (M.dec[hf * 32u + i] * f) * (o[i] + x[i]);
            }
            if (!(ok = wait(DB_M2, c))) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            load32(x, DT_M2 + hf * 32u);
            float f4, most_d = 0.f, most_dk = 0.f;
            {
                const float f[2] = {unit * M.f_t[2u * hf], unit * M.f_t[2u * hf + 1u]};
#pragma unroll
                for (uint32_t i = 0; i < 32u; ++i) {
                    x[i] *= f[i >> 4]; r[i] = x[i] * M.kdec[hf * 32u + i];
                    most_d = fmaxf(most_d, fabsf(x[i])); most_dk = fmaxf(most_dk, fabsf(r[i]));
                }
                s_ex[3][hf][j] = most_d;
                most_dk = both(most_dk, 0u);
                if (!ok) break;
                most_d = fmaxf(most_d, s_ex[3][hf ^ 1u][j]);
                dc_scale(most_dk, up, f4);
                dc_put32(r, up, mine + DT_DK + hf * 16u, mine + DT_DK + 32u + hf * 16u);
                dc_hand_over(bar(DB_DK));
                dc_scale(most_d, up, unit);
                dc_put32(x, up, mine + DT_D + hf * 16u, mine + DT_D + 32u + hf * 16u);
                dc_hand_over(bar(DB_D));
                f4 *= M.f_k;                     // of M4's
            }
            const float last = M.last;
            if (!(ok = wait(DB_M4 + hf, c))) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
            for (int i = 0; i < 64; i += 32) {
                load32(x, DT_M4 + hf * 64u + i);
#pragma unroll
                for (int e = 0; e < 32; ++e) s[i + e] = fmaf(x[e], f4, s[i + e] * last);
            }
            nan = from < (uint32_t)DC_T;
            if (c + 1u < chunks) {
                put_s(fminf(last * most_s + 64.f * most_dk * most_k, 3e38f));
                most_s = 0.f;                    // its own largest, for the bounds of the next chunk
#pragma unroll
                for (int i = 0; i < 64; ++i) most_s = fmaxf(most_s, fabsf(s[i]));
            }
            if (!(ok = wait(DB_M3, c) && (c == 0u || wait(DB_OFREE, c - 1u)))) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            load32(x, DT_M3 + hf * 32u);
            const uint32_t bad_q = M.bad_q[hf];
            const float f3[2] = {unit * A.scale * M.f_p[2u * hf], unit * A.scale * M.f_p[2u * hf + 1u]};
#pragma unroll
            for (uint32_t i = 0; i < 32u; ++i) x[i] = fmaf(x[i], f3[i >> 4], A.scale * o[i]);
            if (bad_q || from < (uint32_t)DC_T)
#pragma unroll
                for (uint32_t i = 0; i < 32u; ++i) if (((bad_q >> i) & 1u) || hf * 32u + i >= from) x[i] = NAN;
#pragma unroll
            for (uint32_t i = 0; i < 32u; ++i) s_out[(hf * 32u + i) * DC_S + j] = from_f32<T>(x[i]);
            __syncwarp();
            if (lane == 0u) tc_arrive(bar(DB_OUT));
        }
        if (ok) {                                // every product has been waited for: the operands' shared memory is free
#pragma unroll
            for (int i = 0; i < 16; ++i)
                *reinterpret_cast<float4 *>(sm + j * DC_SROW + hf * 256u + i * 16u) = nan ? make_float4(NAN, NAN, NAN, NAN) : make_float4(s[4 * i], s[4 * i + 1], s[4 * i + 2], s[4 * i + 3]);
            __syncwarp();
            if (lane == 0u) tc_arrive(bar(DB_END));
            if (wait(DB_END, 0u))
#pragma unroll
                for (int i = 0; i < 16; ++i) *reinterpret_cast<float4 *>(state + (i * 8u + warp) * DC_S + lane * 4u) = *reinterpret_cast<const float4 *>(sm + (i * 8u + warp) * DC_SROW + lane * 16u);
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (fail && tid == 0u && A.status) A.status[ST_TIMEOUT] = 1u;
    if (warp == DC_CONTROL) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(512u) : "memory");
}

// ---- few states: 32 rows a block -------------------------------------------------------------------------------------------------------------------
// The same products the other way round, so that a state is worked on by four blocks: tokens or the state's columns are the 128 lanes of tensor memory, a block's 32 rows (of values) the columns.
//     M1  [K | Q] S^T      M2  [T | P] R      M4  K^T D'      M3  [T | P] D
// Lanes 0 to 63 of M1 and M2 become R and D, lanes 64 to 127 of M1 and M3 the outputs; warps 0, 1, 4 and 5 make the former, 2, 3, 6 and 7 the latter, all of them the state (16 rows a thread). The operands A come
// as k_delta_prep left them, T and P by two warps of their own, row block by row block as far as the triangles reach. R, D, D' and S are operands B in shared memory, which the threads write as [row / 8][k][8 rows]. Their digits have
// one exponent for the block's 32 rows: a row 2^17 smaller than the largest keeps its 22 bits. Bounds, truncation and what is not finite as above.
// What bounds it is the same chain with shorter links, some 4800 cycles a chunk (a prompt of 2000 tokens 95 us, 128 blocks): M1 1160, R 890, M2 640, D' 690, M4 820, S 600; a product takes some 65 cycles, whatever its columns, as it reads 4 KB of A.
constexpr int DN_ROWS = 32;
constexpr uint32_t DN_CONTROL = 8u, DN_TP = 9u, DN_THREADS = 352u;             // 9: T, 10: P
enum : uint32_t { NT_M1 = 0, NT_M2 = 128, NT_M3 = 192, NT_M4 = 256, NT_COLS = 512 };     // each 32 columns for the upper digits' products and 32 for those with a lower digit; M1 twice
enum : uint32_t { NB_KQ, NB_KT, NB_META0, NB_META1, NB_M1, NB_M2, NB_M3, NB_M4, NB_T, NB_P, NB_R, NB_DK, NB_D, NB_Y, NB_Z, NB_S, NB_X, NB_COUNT };
constexpr uint32_t DN_TILE = DC_T * DN_ROWS * 2u, DN_STILE = DC_S * DN_ROWS * 2u, DN_SQ = 2u * DC_SQ;        // a digit of R, D or D'; of S; of T and P together
constexpr uint32_t dn_smem_bytes(int dig) { return dc_keys(dig) + 2u * DN_SQ + 2u * DN_STILE + 6u * DN_TILE + 2u * (uint32_t)sizeof(DcMeta); }
static_assert(dn_smem_bytes(2) <= 224u * 1024u, "shared memory");

// 16 rows' values x f as digits of operand B: two pieces of eight rows, each `piece` bytes after the other; lower digits `low` bytes behind the upper ones
__device__ __forceinline__ void dn_put16(const float (&x)[16], float f, uint8_t *to, uint32_t piece, uint32_t low) {
    uint32_t h[8], l[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float2 y = __fmul2_rn(make_float2(x[2 * i], x[2 * i + 1]), make_float2(f, f));
        dc_digits(y.x, y.y, h[i], l[i]);
    }
#pragma unroll
    for (uint32_t p = 0; p < 2u; ++p) {
        *reinterpret_cast<uint4 *>(to + p * piece) = make_uint4(h[4u * p], h[4u * p + 1u], h[4u * p + 2u], h[4u * p + 3u]);
        *reinterpret_cast<uint4 *>(to + p * piece + low) = make_uint4(l[4u * p], l[4u * p + 1u], l[4u * p + 2u], l[4u * p + 3u]);
    }
}
// what a warp has written to shared memory for the tensor cores, and read from tensor memory, is done with
__device__ __forceinline__ void dn_hand_over(uint32_t mbar) {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncwarp();
    if ((threadIdx.x & 31u) == 0u) tc_arrive(mbar);
}
// the largest number there is (infinities and NaN are none)
__device__ __forceinline__ float dn_most(const float (&x)[16]) {
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) { const float a = fabsf(x[i]); most = fmaxf(most, a < INFINITY ? a : 0.f); }
    return dc_warp_max(most);
}

template <class T, int DIG>
__global__ void __launch_bounds__(DN_THREADS, 1) k_delta_chunk_rows(DeltaArgs A, uint32_t n_seqs, const uint8_t *ws, uint64_t slots, const DcSeq *plan) {
    pdl_prologue();
    constexpr uint32_t KEYS = dc_keys(DIG), SPLIT = DC_S / DN_ROWS;
    extern __shared__ __align__(128) uint8_t sm[];
    __shared__ __align__(8) uint64_t s_bar[NB_COUNT];
    __shared__ float s_mv[2][4], s_mr[2][4], s_md[2][4], s_ms[2][8], s_unit[2][2];
    __shared__ uint32_t s_from[4][DN_ROWS], tmem_slot;       // first tokens from which a row is no number (64: none), of a chunk in turn
    __shared__ volatile uint32_t fail;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const uint32_t h = blockIdx.x / SPLIT, n0 = blockIdx.x % SPLIT * DN_ROWS, kh = h / (A.rank / A.groups);
    __shared__ DcSeq seq;
    dc_seq(A, n_seqs, plan, blockIdx.y, seq);
    const int32_t lo = seq.lo, hi = seq.hi;
    if (lo < 0 || hi < lo || (uint32_t)hi > A.n_tokens) { if (A.status && tid == 0u) A.status[ST_SEQ_BOUNDS] = 1u; return; }
    const int32_t state_slot = delta_slot(A.slots, A.n_slots, seq.b, A.status);
    if (state_slot < 0 || lo == hi) return;
    const uint32_t chunks = ((uint32_t)(hi - lo) + DC_T - 1u) / DC_T;
    const uint64_t slot0 = seq.first;
    if (slot0 + chunks > slots) { if (A.status && tid == 0u) A.status[ST_SEQ_BOUNDS] = 1u; return; }
    uint8_t *const s_kq = sm, *const s_kt = sm + DIG * DC_KQ, *const s_tp = sm + KEYS, *const s_s = s_tp + 2u * DN_SQ, *const s_r = s_s + 2u * DN_STILE, *const s_d = s_r + 2u * DN_TILE, *const s_dk = s_d + 2u * DN_TILE,
                  *const s_meta = s_dk + 2u * DN_TILE;
    const uint8_t *const key = ws + (slot0 * A.groups + kh) * KEYS, *const rec = ws + slots * A.groups * KEYS + (slot0 * A.rank + h) * DC_REC;
    const uint64_t key_step = (uint64_t)A.groups * KEYS, rec_step = (uint64_t)A.rank * DC_REC;
    auto bar = [&](uint32_t i) { return dc_smem(&s_bar[i]); };
    if (tid == 0u) {
        fail = 0u;
        for (uint32_t i = 0; i < NB_COUNT; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(bar(i)), "r"(i >= NB_S ? 8u : i >= NB_R ? 4u : 1u));
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (tid < 4u * DN_ROWS) s_from[tid / DN_ROWS][tid % DN_ROWS] = DC_T;
    if (warp == DN_CONTROL) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(dc_smem(&tmem_slot)), "r"((uint32_t)NT_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0), fail_at = dc_smem(const_cast<uint32_t *>(&fail));
    auto wait = [&](uint32_t i, uint32_t parity) { return tc_wait(bar(i), parity & 1u, fail_at); };

    if (warp == DN_CONTROL) {
        const uint32_t leader = tc_elect();
        auto expect = [&](uint32_t i, uint32_t bytes) { asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" :: "r"(bar(i)), "r"(bytes) : "memory"); };
        auto copy = [&](uint32_t i, const void *dst, const void *src, uint32_t bytes) {
            if (lane) return;
            expect(i, bytes);
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" :: "r"(dc_smem(dst)), "l"(src), "r"(bytes), "r"(bar(i)) : "memory");
        };
        auto get_kq = [&](uint32_t c) { copy(NB_KQ, s_kq, key + c * key_step, DIG * DC_KQ); };
        auto get_kt = [&](uint32_t c) { copy(NB_KT, s_kt, key + c * key_step + DIG * DC_KQ, DIG * DC_KT); };
        auto get_meta = [&](uint32_t c) { copy(NB_META0 + (c & 1u), s_meta + (c & 1u) * sizeof(DcMeta), rec + c * rec_step + 4u * DC_SQ, sizeof(DcMeta)); };
        get_meta(0u); get_kq(0u); get_kt(0u);
        const uint64_t a_kq = tc_smem_desc(dc_smem(s_kq), 2048u, 128u), a_kt = tc_smem_desc(dc_smem(s_kt), 2048u, 128u), a_tp = tc_smem_desc(dc_smem(s_tp), 2048u, 128u);
        // operands B: 128 bytes from eight k to the next, a piece from eight rows to the next
        const uint64_t b_s = tc_smem_desc(dc_smem(s_s), 128u, DC_S * 16u), b_r = tc_smem_desc(dc_smem(s_r), 128u, DC_T * 16u), b_d = tc_smem_desc(dc_smem(s_d), 128u, DC_T * 16u), b_dk = tc_smem_desc(dc_smem(s_dk), 128u, DC_T * 16u);
        const uint32_t both = tc_idesc(2u * DN_ROWS) | (1u << 16), one = tc_idesc(DN_ROWS) | (1u << 16);     // B with the rows, not k, next to one another
        // results = A B^T over 64 of k: A's upper digits with both of B's at once (a product reads 4 KB of A, which takes longer than its operations), then its lower ones, a_lo 16-byte units behind, with B's upper ones
        auto product = [&](uint32_t d, uint64_t a, uint32_t a_lo, bool a_two, uint64_t bd) {
#pragma unroll
            for (uint32_t k = 0; k < 4u; ++k) tc_mma_if(leader, tmem + d, a + k * 256u, bd + k * 16u, both, k ? 1u : 0u);
            if (a_two)
#pragma unroll
                for (uint32_t k = 0; k < 4u; ++k) tc_mma_if(leader, tmem + d + DN_ROWS, a + a_lo + k * 256u, bd + k * 16u, one, 1u);
        };
        uint32_t c = 0u;
#pragma unroll 1
        for (; c < chunks; ++c) {
            const bool more = c + 1u < chunks;
            if (!wait(NB_KQ, c) || !wait(NB_S, c)) break;        // the one that comes last goes last: a wait takes its time also for what is there
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            product(NT_M1, a_kq, DC_KQ >> 4, DIG == 2, b_s);
            product(NT_M1 + 64u, a_kq + 4u * 256u, DC_KQ >> 4, DIG == 2, b_s + 4u * 16u);
            tc_commit_if(leader, bar(NB_M1));
            if (c) { if (!wait(NB_M4, c - 1u)) break; get_kt(c); }
            if (!wait(NB_M1, c)) break;
            if (more) get_kq(c + 1u);
            if (!wait(NB_T, c) || !wait(NB_P, c) || !wait(NB_R, c)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            product(NT_M2, a_tp, DN_SQ >> 4, true, b_r);
            tc_commit_if(leader, bar(NB_M2));
            if (more) get_meta(c + 1u);
            if (!wait(NB_KT, c) || !wait(NB_DK, c)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            product(NT_M4, a_kt, DC_KT >> 4, DIG == 2, b_dk);
            tc_commit_if(leader, bar(NB_M4));
            if (!wait(NB_D, c)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            product(NT_M3, a_tp, DN_SQ >> 4, true, b_d);
            tc_commit_if(leader, bar(NB_M3));
        }
        if (!fail) wait(NB_M3, chunks - 1u);
        // where a wait was given up, copies that nobody waits for may still be writing into this block's shared memory: every stage is waited for in both its phases
        if (fail && lane == 0u) for (uint32_t i = NB_KQ; i <= NB_META1; ++i) { mbar_wait(bar(i), 0u); mbar_wait(bar(i), 1u); }
    } else if (warp >= DN_TP) {                  // T to the upper 64 rows of [k / 8][row][8 of k], P to the lower ones; what lies above a diagonal block of 16 is zero throughout
        const uint32_t part = warp - DN_TP;
        uint8_t *const to = s_tp + part * (DC_T * 16u);
        for (uint32_t i = lane; i < 2u * 8u * DC_T; i += 32u) {
            const uint32_t d = i / (8u * DC_T), piece = i / DC_T % 8u, row = i % DC_T;
            if (row / 16u < piece / 2u) *reinterpret_cast<uint4 *>(to + d * DN_SQ + piece * 2048u + row * 16u) = make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll 1
        for (uint32_t c = 0; c < chunks; ++c) {
            if (c && !wait(NB_M3, c - 1u)) break;
            const uint8_t *const from = rec + c * rec_step + part * 2u * DC_SQ;
#pragma unroll
            for (uint32_t piece = 0; piece < 8u; ++piece)
#pragma unroll
                for (uint32_t r = 0; r < DC_T; r += 32u) {
                    const uint32_t row = r + lane;
                    if (row / 16u >= piece / 2u)
#pragma unroll
                        for (uint32_t d = 0; d < 2u; ++d)
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(dc_smem(to) + d * DN_SQ + piece * 2048u + row * 16u), "l"(from + d * DC_SQ + dc_sq_at(row, piece)) : "memory");
                }
            asm volatile("cp.async.wait_all;" ::: "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0u) tc_arrive(bar(NB_T + part));
        }
    } else {
        const uint32_t w = warp & 3u, hf = warp >> 2, mine = tmem + ((w * 32u) << 16), at = hf * 16u, half = w & 1u, t = half * 32u + lane;       // t: the thread's token
        const bool rows = w < 2u;                // makes R and D, else outputs
        const uint32_t me = hf * 2u + half;      // among the four warps of a kind
        bool ok = true;
        auto load16 = [&](float (&x)[16], uint32_t col) {
            uint32_t y[16], z[16];
            dc_ld16(y, mine + col + at);
            dc_ld16(z, mine + col + DN_ROWS + at);
            dc_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = __uint_as_float(y[i]) + __uint_as_float(z[i]);
        };
        auto load_m1 = [&](float (&x)[16]) {
            uint32_t y[4][16];
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i) dc_ld16(y[i], mine + NT_M1 + i * 32u + at);
            dc_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = (__uint_as_float(y[0][i]) + __uint_as_float(y[2][i])) + (__uint_as_float(y[1][i]) + __uint_as_float(y[3][i]));
        };
        float *const state = A.state + (((uint64_t)(uint32_t)state_slot * A.rank + h) * DC_S + n0 + at) * DC_S + w * 32u + lane;         // rows at .. at + 15 of the block, column w 32 + lane
        float s[16], v[16], up, unit_s;
        uint32_t nan = 0u;                       // rows that are no numbers any more, as bits
        auto put_s = [&](float bound) {
            dc_scale(bound, up, unit_s);
            dn_put16(s, up, s_s + hf * 2u * (DC_S * 16u) + (w * 32u + lane) * 16u, DC_S * 16u, DN_STILE);
            dn_hand_over(bar(NB_S));
        };
        // The largest of the warp's part of the state, for the bounds of chunk c; a row that is not finite is no number from that chunk on
        auto look_at_s = [&](uint32_t c) {
            const float most = dn_most(s);
            bool odd = false;
#pragma unroll
            for (int i = 0; i < 16; ++i) odd |= !(fabsf(s[i]) < INFINITY);
            if (odd)
#pragma unroll
                for (int i = 0; i < 16; ++i) if (!(fabsf(s[i]) < INFINITY)) { s[i] = 0.f; atomicMin(&s_from[c & 3u][at + i], 0u); }
            __syncwarp();
            if (lane == 0u) s_ms[c & 1u][warp] = most;
        };
        const T *const vp = reinterpret_cast<const T *>(A.v) + (uint64_t)(uint32_t)lo * A.v_stride + (uint64_t)h * DC_S + n0 + at;
        auto get_v = [&](uint32_t c) {           // of the thread's token of chunk c
            const uint32_t i = c * DC_T + t;
            constexpr int N = 16 / sizeof(T);
#pragma unroll
            for (int e = 0; e < 16; e += N) {
                float y[N];
#pragma unroll
                for (int j = 0; j < N; ++j) y[j] = 0.f;
                if (rows && i < (uint32_t)(hi - lo)) load_vals<N>(vp + (uint64_t)i * A.v_stride + e, y);
#pragma unroll
                for (int j = 0; j < N; ++j) v[e + j] = y[j];
            }
        };
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = state[i * DC_S];
        get_v(0u);
        look_at_s(0u);
        asm volatile("bar.sync 1, 256;" ::: "memory");         // all eight warps come here
        {
            float most = s_ms[0][0];
#pragma unroll
            for (int i = 1; i < 8; ++i) most = fmaxf(most, s_ms[0][i]);
            put_s(most);
        }
#pragma unroll 1
        for (uint32_t c = 0; ok && c < chunks; ++c) {
            const DcMeta &M = *reinterpret_cast<const DcMeta *>(s_meta + (c & 1u) * sizeof(DcMeta));
            float x[16], o[16], unit, unit_d, unit_dk, most_v = 0.f;
            if (rows) {                          // the chunk's values
                bool odd = false;
#pragma unroll
                for (int i = 0; i < 16; ++i) odd |= !(fabsf(v[i]) < INFINITY);
                if (odd)
#pragma unroll
                    for (int i = 0; i < 16; ++i) if (!(fabsf(v[i]) < INFINITY)) { v[i] = 0.f; atomicMin(&s_from[c & 3u][at + i], t); }
                most_v = dn_most(v);
                if (lane == 0u) s_mv[c & 1u][me] = most_v;
            }
            __syncwarp();
            if (lane == 0u) tc_arrive(bar(NB_X));
            if (!(ok = wait(NB_META0 + (c & 1u), c >> 1) && wait(NB_X, c))) break;
            float most_s = s_ms[c & 1u][0];
#pragma unroll
            for (int i = 1; i < 8; ++i) most_s = fmaxf(most_s, s_ms[c & 1u][i]);
            const uint32_t from = lane >= 16u ? (uint32_t)DC_T : (nan >> lane) & 1u ? 0u : min(M.nan_from, s_from[c & 3u][at + lane]);       // of row at + lane
            nan = __ballot_sync(0xffffffffu, from < (uint32_t)DC_T);
            const float most_k = 32768.f * M.f_k, dec = M.dec[t];        // no key is larger
            if (rows) {
#pragma unroll
                for (int i = 0; i < 4; ++i) most_v = fmaxf(most_v, s_mv[c & 1u][i]);
                dc_scale(fminf(most_v + M.most_dec * (128.f * most_s) * most_k, 3e38f), up, unit);
                if (!(ok = wait(NB_M1, c))) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                load_m1(x);
                const float f = -(unit_s * M.f_k) * dec;
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] = fmaf(f, x[i], v[i]);
                uint8_t *const mine_b = s_r + hf * 2u * (DC_T * 16u) + t * 16u;
                dn_put16(x, up, mine_b, DC_T * 16u, DN_TILE);
                dn_hand_over(bar(NB_R));
                const float most_r = dn_most(x);
                if (lane == 0u) s_mr[c & 1u][me] = most_r;
                __syncwarp();
                if (lane == 0u) tc_arrive(bar(NB_Y));
                if (half == 0u && lane < 16u) s_from[(c + 2u) & 3u][at + lane] = DC_T;       // what chunk c - 2 left there was read ahead of NB_X
                get_v(c + 1u);
                const float f2 = unit * M.f_t[t >> 4], kdec = M.kdec[t];
                if (!(ok = wait(NB_Y, c))) break;
                // no D is larger than the largest R times the largest row of T
                const float most_d = fminf(fmaxf(fmaxf(s_mr[c & 1u][0], s_mr[c & 1u][1]), fmaxf(s_mr[c & 1u][2], s_mr[c & 1u][3])) * fmaxf(fmaxf(M.t_sum[0], M.t_sum[1]), fmaxf(M.t_sum[2], M.t_sum[3])), 3e38f);
                float up_d;
                dc_scale(most_d, up_d, unit_d);
                dc_scale(fminf(most_d * M.most_kdec, 3e38f), up, unit_dk);
                if (lane == 0u) { s_unit[c & 1u][0] = unit_d; s_unit[c & 1u][1] = unit_dk; }         // of all four warps the same
                if (!(ok = wait(NB_M2, c))) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                load16(x, NT_M2);
#pragma unroll
                for (int i = 0; i < 16; ++i) { x[i] *= f2; o[i] = x[i] * kdec; }
                dn_put16(o, up, s_dk + hf * 2u * (DC_T * 16u) + t * 16u, DC_T * 16u, DN_TILE);
                dn_hand_over(bar(NB_DK));
                dn_put16(x, up_d, s_d + hf * 2u * (DC_T * 16u) + t * 16u, DC_T * 16u, DN_TILE);
                dn_hand_over(bar(NB_D));
                const float most_dk = dn_most(o);
                if (lane == 0u) s_md[c & 1u][me] = most_dk;
                __syncwarp();
                if (lane == 0u) tc_arrive(bar(NB_Z));
            } else {
                if (!(ok = wait(NB_M1, c))) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                load_m1(o);
                const float f = (unit_s * M.f_q) * dec * A.scale;
#pragma unroll
                for (int i = 0; i < 16; ++i) o[i] *= f;
            }
            if (!(ok = wait(NB_Z, c))) break;
            const float most_dk = fmaxf(fmaxf(s_md[c & 1u][0], s_md[c & 1u][1]), fmaxf(s_md[c & 1u][2], s_md[c & 1u][3]));
            if (!rows) { unit_d = s_unit[c & 1u][0]; unit_dk = s_unit[c & 1u][1]; }
            const float f4 = unit_dk * M.f_k, last = M.last, f3 = unit_d * A.scale * M.f_p[t >> 4];
            const bool bad_q = (M.bad_q[half] >> lane) & 1u;
            if (!(ok = wait(NB_M4, c))) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            load16(x, NT_M4);
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = fmaf(x[i], f4, s[i] * last);
            if (c + 1u < chunks) {
                put_s(fminf(last * most_s + 64.f * most_dk * most_k, 3e38f));
                look_at_s(c + 1u);
            }
            if (rows) continue;
            if (!(ok = wait(NB_M3, c))) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            load16(x, NT_M3);
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = fmaf(x[i], f3, o[i]);
            if (nan || __any_sync(0xffffffffu, bad_q))
#pragma unroll
                for (int i = 0; i < 16; ++i) if (bad_q | (t >= __shfl_sync(0xffffffffu, from, i))) x[i] = NAN;
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            const uint32_t token = c * DC_T + t;
            if (token < (uint32_t)(hi - lo)) {
                constexpr int N = 16 / sizeof(T);
                T *const out = reinterpret_cast<T *>(A.out) + ((uint64_t)((uint32_t)lo + token) * A.rank + h) * DC_S + n0 + at;
#pragma unroll
                for (int e = 0; e < 16; e += N) {
                    float y[N];
#pragma unroll
                    for (int j = 0; j < N; ++j) y[j] = x[e + j];
                    store_vals<N>(out + e, y);
                }
            }
        }
        if (ok)
#pragma unroll
            for (int i = 0; i < 16; ++i) state[i * DC_S] = (nan >> i) & 1u ? NAN : s[i];
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (fail && tid == 0u && A.status) A.status[ST_TIMEOUT] = 1u;
    if (warp == DN_CONTROL) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"((uint32_t)NT_COLS) : "memory");
}

static uint64_t dc_records(int dig, uint32_t groups, uint32_t rank, uint64_t slots) { return slots * ((uint64_t)groups * dc_keys(dig) + (uint64_t)rank * DC_REC); }
uint64_t delta_chunk_workspace(uint32_t type, uint32_t groups, uint32_t rank, uint32_t n_tokens, uint32_t n_seqs) {
    return dc_records(type == VT_F32 ? 2 : 1, groups, rank, dc_slots(n_tokens, n_seqs)) + (n_seqs > DC_NEAR ? n_seqs * (sizeof(DcSeq) + 4ull) : 0u);
}

template <class T, int DIG> static int launch_chunk(DeltaArgs A, uint32_t n_seqs, const uint8_t *ws, uint64_t slots, const DcSeq *plan, cudaStream_t s) {
    // Four blocks a state where that gives no multiprocessor two, and sequences of four chunks on the average: 32 heads, 1 sequence of 64 tokens 25.6 -> 27.5 us in F32 (21.5 -> 21.0 in BF16), of 128 30 -> 34 (24 -> 27), of 256
    // 40 -> 41 (33 -> 32), of 500 56 -> 52 (49 -> 43), of 2000 172 -> 136 (156 -> 131), of 8000 606 -> 519 (561 -> 482), each with the preparation. In two turns four blocks would take 5.5 us a chunk, one takes 4.
    if ((uint64_t)A.rank * n_seqs * (DC_S / DN_ROWS) <= sm_count() && A.n_tokens >= 256u * (uint64_t)n_seqs) {
        static std::atomic<uint64_t> set_rows{0};
        if (!raise_smem_limit(reinterpret_cast<const void *>(k_delta_chunk_rows<T, DIG>), dn_smem_bytes(DIG), set_rows)) return 0;
        RC_LAUNCH((k_delta_chunk_rows<T, DIG>), dim3(A.rank * (DC_S / DN_ROWS), n_seqs), DN_THREADS, dn_smem_bytes(DIG), s, A, n_seqs, ws, slots, plan);
        RC_LAUNCHED();
        return 1;
    }
    static std::atomic<uint64_t> set{0};
    if (!raise_smem_limit(reinterpret_cast<const void *>(k_delta_chunk<T, DIG>), dc_smem_bytes(DIG, sizeof(T)), set)) return 0;
    for (uint32_t b = 0; b < n_seqs; b += 65535u) {
        A.first_seq = b;
        RC_LAUNCH((k_delta_chunk<T, DIG>), dim3(A.rank, n_seqs - b < 65535u ? n_seqs - b : 65535u), DC_THREADS, dc_smem_bytes(DIG, sizeof(T)), s, A, n_seqs, ws, slots, plan);
        RC_LAUNCHED();
    }
    return 1;
}
template <class T, int DIG> static int launch_chunks(const DeltaArgs &A, uint32_t n_seqs, uint8_t *ws, cudaStream_t s) {
    const uint64_t slots = dc_slots(A.n_tokens, n_seqs);
    constexpr size_t smem = 4u * DC_MAT > DIG * DC_KQ ? 4u * DC_MAT : DIG * DC_KQ;
    RC_REQUIRE(slots <= 0x7fffffffu && A.groups <= 65535u, "delta rule: too many chunks");
    DcSeq *const plan = (DcSeq *)(ws + dc_records(DIG, A.groups, A.rank, slots));
    prof_begin("delta_prep", s);
    if (n_seqs > DC_NEAR) {
        RC_LAUNCH(k_delta_plan, 1, 1024, 0, s, A, n_seqs, plan);
        RC_LAUNCHED();
    }
    if (A.rank > 2u * A.groups) {
        static std::atomic<uint64_t> set{0};
        if (!raise_smem_limit(reinterpret_cast<const void *>(k_delta_prep<T, DIG, true>), smem, set)) return 0;
        RC_LAUNCH((k_delta_prep<T, DIG, true>), dim3((uint32_t)slots, A.groups), 256, smem, s, A, n_seqs, ws, slots, plan);
    } else {
        static std::atomic<uint64_t> set{0};
        if (!raise_smem_limit(reinterpret_cast<const void *>(k_delta_prep<T, DIG, false>), smem, set)) return 0;
        RC_LAUNCH((k_delta_prep<T, DIG, false>), dim3((uint32_t)slots, A.groups), 256, smem, s, A, n_seqs, ws, slots, plan);
    }
    RC_LAUNCHED();
    prof_end(s);
    prof_begin("delta_chunk", s);
    const int ok = launch_chunk<T, DIG>(A, n_seqs, ws, slots, plan, s);
    prof_end(s);
    return ok;
}

int launch_delta_chunks(const DeltaArgs &A, uint32_t type, uint32_t n_seqs, uint8_t *ws, cudaStream_t s) {
    return type == VT_F32 ? launch_chunks<float, 2>(A, n_seqs, ws, s) : type == VT_F16 ? launch_chunks<__half, 1>(A, n_seqs, ws, s) : launch_chunks<__nv_bfloat16, 1>(A, n_seqs, ws, s);
}

}  // namespace rc
