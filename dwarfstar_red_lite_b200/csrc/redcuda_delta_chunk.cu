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

#include <math.h>

namespace rc {

constexpr int DC_T = 64, DC_S = 128;             // tokens of a chunk; the state
constexpr uint32_t DC_TILE = DC_T * DC_S * 2u;   // a digit of the chunk's keys or queries: [token][128] with the 16-byte pieces of a row turned by its number
constexpr uint32_t DC_SQ = DC_T * DC_T * 2u;     // a digit of T or P: [t][s], likewise
struct DcMeta {                                  // of a chunk and value head
    float dec[DC_T], kdec[DC_T];                 // exp(G_t), exp(G_last - G_t)
    float last, f_k, f_q, f_t, f_p;              // exp(G_last); what a digit's unit is worth in K, Q, T, P
    uint32_t nan_from, bad_q[2], pad[120];       // tokens from which on everything is NaN; tokens whose query is not finite
};
static_assert(sizeof(DcMeta) == 1024, "copied in whole");
constexpr uint32_t DC_REC = 4u * DC_SQ + (uint32_t)sizeof(DcMeta);       // T hi, T lo, P hi, P lo, meta
__host__ __device__ constexpr uint32_t dc_keys(int dig) { return 2u * (uint32_t)dig * DC_TILE; }      // K hi (, K lo), Q hi (, Q lo)

// Chunks are numbered so that a sequence finds its own without the lengths of the others: chunk c of sequence b is number cu[b] / 64 + b + c.
static uint64_t dc_slots(uint32_t n_tokens, uint32_t n_seqs) { return (uint64_t)n_tokens / DC_T + n_seqs; }

__device__ __forceinline__ uint32_t dc_tile_at(uint32_t t, uint32_t piece) { return t * 256u + (piece ^ (t & 7u)) * 16u; }
__device__ __forceinline__ uint32_t dc_sq_at(uint32_t t, uint32_t piece) { return t * 128u + (piece ^ (t & 7u)) * 16u; }
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
    const float2 h = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
    lo = dc_pack(a - h.x, b - h.y);
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
// A block per chunk and key head: digits of K and Q, K K^T and Q K^T on the tensor cores (their lower triangles), then for each of the key head's value heads (two at a time, half a block
// each) the decays, the inverse of 1 + A and the digits of T and P. The inverse goes by blocks of 16: those on the diagonal by substitution, a column a lane; the others T_ij = -T_ii sum_k A_ik T_kj
// in the order of their distance from it, which is as stable as substitution (powers of A are not, where keys are alike).
constexpr uint32_t DC_PITCH = 68u;               // floats of a row of the 64 x 64 matrices in shared memory
constexpr uint32_t DC_MAT = DC_T * DC_PITCH * 4u;
__device__ __forceinline__ void dc_half_sync(uint32_t half) { asm volatile("bar.sync %0, 128;" :: "r"(half + 1u) : "memory"); }
// the largest over half a block; s: four floats of its own
__device__ __forceinline__ float dc_half_max(float x, float *s, uint32_t half) {
    for (int w = 16; w; w >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, w));
    if ((threadIdx.x & 31u) == 0u) s[(threadIdx.x >> 5) & 3u] = x;
    dc_half_sync(half);
    x = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
    dc_half_sync(half);
    return x;
}

template <class T, int DIG>
__global__ void __launch_bounds__(256, 2) k_delta_prep(DeltaArgs A, uint32_t n_seqs, uint8_t *ws, uint64_t slots) {
    pdl_prologue();
    extern __shared__ __align__(128) uint8_t sm[];
    float *const s_kk = reinterpret_cast<float *>(sm), *const s_qk = s_kk + DC_T * DC_PITCH;
    uint8_t *const dig = sm + 2u * DC_MAT;       // the digits; later the halves' matrices A and T
    __shared__ float s_red[2][8], s_max[2][4], s_beta[2][DC_T];
    __shared__ double s_cum[2][DC_T];
    __shared__ uint32_t s_bad[2][2];             // tokens whose key or query is not finite
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, kh = blockIdx.y, width = A.rank / A.groups;
    const uint64_t slot = blockIdx.x;
    // the sequence: the last b with cu[b] / 64 + b <= slot
    uint32_t b = 0u, cnt = n_seqs;
    while (cnt > 1u) {
        const uint32_t step = (cnt + 31u) / 32u, i = lane * step;
        const bool le = i < cnt && (int64_t)(A.cu[b + i] / DC_T) + (int64_t)(b + i) <= (int64_t)slot;
        const uint32_t m = __ballot_sync(0xffffffffu, le), at = (m ? 31u - (uint32_t)__clz((int)m) : 0u) * step;
        cnt = min(step, cnt - at); b += at;
    }
    const int32_t lo = A.cu[b], hi = A.cu[b + 1u];
    if (lo < 0 || hi < lo || (uint32_t)hi > A.n_tokens) return;          // reported by k_delta_chunk
    const int64_t chunk = (int64_t)slot - (int64_t)(lo / DC_T) - (int64_t)b;
    if (chunk < 0 || chunk * DC_T >= hi - lo) return;
    const uint32_t t0 = (uint32_t)lo + (uint32_t)chunk * DC_T, n = min((uint32_t)DC_T, (uint32_t)hi - t0);

    // rows 8 warp .. 8 warp + 7 of K and Q, four values a lane
    float kx[8][4], qx[8][4], mk = 0.f, mq = 0.f;
    if (tid < 4u) s_bad[tid >> 1][tid & 1u] = 0u;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        const uint32_t t = warp * 8u + r;
        float mr = 0.f, mr2 = 0.f;
        bool fk = true, fq = true;
        if (t < n) {
            load_vals<4>(reinterpret_cast<const T *>(A.k) + (uint64_t)(t0 + t) * A.k_stride + (uint64_t)kh * DC_S + lane * 4u, kx[r]);
            load_vals<4>(reinterpret_cast<const T *>(A.q) + (uint64_t)(t0 + t) * A.q_stride + (uint64_t)kh * DC_S + lane * 4u, qx[r]);
#pragma unroll
            for (int i = 0; i < 4; ++i) { fk &= fabsf(kx[r][i]) < INFINITY; fq &= fabsf(qx[r][i]) < INFINITY; mr = fmaxf(mr, fabsf(kx[r][i])); mr2 = fmaxf(mr2, fabsf(qx[r][i])); }
        }
        const bool ak = __all_sync(0xffffffffu, fk), aq = __all_sync(0xffffffffu, fq);
        if (t >= n || !ak) { mr = 0.f; for (int i = 0; i < 4; ++i) kx[r][i] = 0.f; }
        if (t >= n || !aq) { mr2 = 0.f; for (int i = 0; i < 4; ++i) qx[r][i] = 0.f; }
        if (lane == 0u && !ak) atomicOr(&s_bad[0][t >> 5], 1u << (t & 31u));
        if (lane == 0u && !aq) atomicOr(&s_bad[1][t >> 5], 1u << (t & 31u));
        mk = fmaxf(mk, mr); mq = fmaxf(mq, mr2);
    }
    for (int w = 16; w; w >>= 1) { mk = fmaxf(mk, __shfl_xor_sync(0xffffffffu, mk, w)); mq = fmaxf(mq, __shfl_xor_sync(0xffffffffu, mq, w)); }
    if (lane == 0u) { s_red[0][warp] = mk; s_red[1][warp] = mq; }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) { mk = fmaxf(mk, s_red[0][i]); mq = fmaxf(mq, s_red[1][i]); }
    float up_k, f_k, up_q, f_q;
    dc_scale(mk, up_k, f_k);
    dc_scale(mq, up_q, f_q);
    uint8_t *const keys = ws + (slot * A.groups + kh) * dc_keys(DIG);
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        const uint32_t at = dc_tile_at(warp * 8u + r, lane >> 1) + (lane & 1u) * 8u;
        auto put = [&](const float (&x)[4], float up, uint32_t tile) {
            uint2 h, l;
            dc_digits(x[0] * up, x[1] * up, h.x, l.x);
            dc_digits(x[2] * up, x[3] * up, h.y, l.y);
            *reinterpret_cast<uint2 *>(dig + tile * DC_TILE + at) = h;
            *reinterpret_cast<uint2 *>(keys + tile * DC_TILE + at) = h;
            if (DIG == 2) { *reinterpret_cast<uint2 *>(dig + (tile + 1u) * DC_TILE + at) = l; *reinterpret_cast<uint2 *>(keys + (tile + 1u) * DC_TILE + at) = l; }
        };
        put(kx[r], up_k, 0u);
        put(qx[r], up_q, DIG);
    }
    __syncthreads();
    {   // warps 0-3: K K^T, 4-7: Q K^T; 16 rows each, the columns up to the diagonal
        const uint32_t mt = warp & 3u, which = warp >> 2, a_at = dc_smem(dig) + which * DIG * DC_TILE, b_at = dc_smem(dig);
        const uint32_t ar = mt * 16u + (lane & 15u), ac = lane >> 4, br = (lane & 7u) + (lane >> 4) * 8u, bc = (lane >> 3) & 1u;
        float c[4][2][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) c[i][j][e] = 0.f;
#pragma unroll 2
        for (uint32_t s = 0; s < 8u; ++s) {
            uint32_t ah[4], al[4];
            dc_ldsm(ah, a_at + dc_tile_at(ar, 2u * s + ac));
            if (DIG == 2) dc_ldsm(al, a_at + DC_TILE + dc_tile_at(ar, 2u * s + ac));
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i)
                if (i <= mt) {
                    uint32_t x[4];
                    dc_ldsm(x, b_at + dc_tile_at(i * 16u + br, 2u * s + bc));
                    dc_mma(c[i][0], ah, x[0], x[1]); dc_mma(c[i][1], ah, x[2], x[3]);
                    if (DIG == 2) {
                        dc_mma(c[i][0], al, x[0], x[1]); dc_mma(c[i][1], al, x[2], x[3]);
                        dc_ldsm(x, b_at + DC_TILE + dc_tile_at(i * 16u + br, 2u * s + bc));
                        dc_mma(c[i][0], ah, x[0], x[1]); dc_mma(c[i][1], ah, x[2], x[3]);
                    }
                }
        }
        float *const to = which ? s_qk : s_kk;
        const float f = which ? f_q : f_k;
        const uint32_t g = lane >> 2, c2 = (lane & 3u) * 2u;
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i)
            if (i <= mt)
#pragma unroll
                for (uint32_t j = 0; j < 2u; ++j) {
                    float *p = to + (mt * 16u + g) * DC_PITCH + i * 16u + j * 8u + c2;
                    *reinterpret_cast<float2 *>(p) = make_float2(c[i][j][0] * f * f_k, c[i][j][1] * f * f_k);
                    *reinterpret_cast<float2 *>(p + 8u * DC_PITCH) = make_float2(c[i][j][2] * f * f_k, c[i][j][3] * f * f_k);
                }
    }
    __syncthreads();
    const uint32_t half = tid >> 7, ht = tid & 127u, hw = ht >> 5;
    float *const s_a = reinterpret_cast<float *>(dig + half * 2u * DC_MAT), *const s_t = s_a + DC_T * DC_PITCH;
    float *const s_m = s_max[half];
    for (uint32_t v = half; v < width; v += 2u) {
        const uint32_t h = kh * width + v;
        uint8_t *const rec = ws + slots * A.groups * dc_keys(DIG) + (slot * A.rank + h) * DC_REC;
        DcMeta *const meta = reinterpret_cast<DcMeta *>(rec + 4u * DC_SQ);
        if (hw == 0u) {                          // tokens 2 lane and 2 lane + 1
            double g[2];
            float bt[2];
            bool bad[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t t = lane * 2u + i;
                float gv = 0.f, bv = 0.f;
                if (t < n) { gv = A.gate[(uint64_t)(t0 + t) * A.rank + h]; bv = A.beta[(uint64_t)(t0 + t) * A.rank + h]; }
                gv = gv < -200.f ? -200.f : gv;  // exp is 0 from -104 on; -infinity cuts the past off
                bad[i] = !(gv < INFINITY) || !(fabsf(bv) < INFINITY) || ((s_bad[0][t >> 5] >> (t & 31u)) & 1u);
                g[i] = bad[i] ? 0.0 : (double)gv; bt[i] = bad[i] ? 0.f : bv;
            }
            g[1] += g[0];
            double sum = g[1];
            for (int w = 1; w < 32; w <<= 1) { const double x = __shfl_up_sync(0xffffffffu, sum, w); if (lane >= (uint32_t)w) sum += x; }
            const double before = sum - g[1], last = __shfl_sync(0xffffffffu, sum, 31);
            const uint32_t m0 = __ballot_sync(0xffffffffu, bad[0]), m1 = __ballot_sync(0xffffffffu, bad[1]);
            const uint32_t first0 = m0 ? 2u * ((uint32_t)__ffs((int)m0) - 1u) : (uint32_t)DC_T, first1 = m1 ? 2u * ((uint32_t)__ffs((int)m1) - 1u) + 1u : (uint32_t)DC_T;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t t = lane * 2u + i;
                const double G = before + g[i];
                s_cum[half][t] = G; s_beta[half][t] = bt[i];
                meta->dec[t] = expf((float)G); meta->kdec[t] = expf((float)(last - G));
            }
            if (lane == 0u) {
                meta->last = expf((float)last); meta->f_k = f_k; meta->f_q = f_q;
                meta->nan_from = min(first0, first1); meta->bad_q[0] = s_bad[1][0]; meta->bad_q[1] = s_bad[1][1];
            }
        }
        dc_half_sync(half);
        // A below the diagonal; P and its digits: pieces of eight columns, four a thread
        float p[4][8], most = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t id = ht + i * 128u, t = id >> 3, s0 = (id & 7u) * 8u;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t s = s0 + j;
                p[i][j] = 0.f;
                float a = 0.f;
                if (s <= t) {
                    const float ratio = s == t ? 1.f : expf((float)(s_cum[half][t] - s_cum[half][s]));
                    p[i][j] = s_qk[t * DC_PITCH + s] * ratio;
                    a = s_beta[half][t] * s_kk[t * DC_PITCH + s] * ratio;
                    most = fmaxf(most, fabsf(p[i][j]));
                }
                s_a[t * DC_PITCH + s] = a;
            }
        }
        most = dc_half_max(most, s_m, half);
        float up, unit;
        dc_scale(most, up, unit);
        if (ht == 0u) meta->f_p = unit;
        auto put = [&](const float (&x)[8], float f, uint32_t t, uint32_t piece, uint8_t *to) {
            uint4 h, l;
            dc_digits(x[0] * f, x[1] * f, h.x, l.x); dc_digits(x[2] * f, x[3] * f, h.y, l.y);
            dc_digits(x[4] * f, x[5] * f, h.z, l.z); dc_digits(x[6] * f, x[7] * f, h.w, l.w);
            *reinterpret_cast<uint4 *>(to + dc_sq_at(t, piece)) = h;
            *reinterpret_cast<uint4 *>(to + DC_SQ + dc_sq_at(t, piece)) = l;
        };
#pragma unroll
        for (int i = 0; i < 4; ++i) { const uint32_t id = ht + i * 128u; put(p[i], up, id >> 3, id & 7u, rec + 2u * DC_SQ); }
        // the diagonal blocks of the inverse: warp hw has block hw, lane c column c
        {
            const uint32_t o = hw * 16u, c = lane & 15u;
            float x[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                float e = (uint32_t)r == c ? 1.f : 0.f;
#pragma unroll
                for (int k = 0; k < r; ++k) e = fmaf(-s_a[(o + r) * DC_PITCH + o + k], x[k], e);
                x[r] = e;
            }
            if (lane < 16u)
#pragma unroll
                for (int r = 0; r < 16; ++r) s_t[(o + r) * DC_PITCH + o + c] = x[r];
        }
        dc_half_sync(half);
        // the others: 64 threads a block, a row and four columns each; first M = sum_k A_ik T_kj, kept where T_ij will be, then -T_ii M
        const uint32_t br = (ht & 63u) >> 2, bc = (ht & 3u) * 4u;
#pragma unroll 1
        for (uint32_t d = 1; d < 4u; ++d)
#pragma unroll 1
            for (uint32_t first = 0; first < 4u - d; first += 2u) {
                const uint32_t j = first + (ht >> 6), i = j + d;
                const bool on = i < 4u;
                float4 m = make_float4(0.f, 0.f, 0.f, 0.f);
                auto fma4 = [&](float a, const float *t) { const float4 y = *reinterpret_cast<const float4 *>(t); m.x = fmaf(a, y.x, m.x); m.y = fmaf(a, y.y, m.y); m.z = fmaf(a, y.z, m.z); m.w = fmaf(a, y.w, m.w); };
                float *const at = s_t + (i * 16u + br) * DC_PITCH + j * 16u + bc;
                if (on) {
#pragma unroll 8
                    for (uint32_t k = j * 16u; k < i * 16u; ++k) fma4(s_a[(i * 16u + br) * DC_PITCH + k], s_t + k * DC_PITCH + j * 16u + bc);
                    *reinterpret_cast<float4 *>(at) = m;
                }
                dc_half_sync(half);
                m = make_float4(0.f, 0.f, 0.f, 0.f);
                if (on) {
#pragma unroll
                    for (uint32_t k = 0; k < 16u; ++k) fma4(-s_t[(i * 16u + br) * DC_PITCH + i * 16u + k], s_t + (i * 16u + k) * DC_PITCH + j * 16u + bc);
                }
                dc_half_sync(half);
                if (on) *reinterpret_cast<float4 *>(at) = m;
                dc_half_sync(half);
            }
        most = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t id = ht + i * 128u, t = id >> 3, s0 = (id & 7u) * 8u;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t s = s0 + j;
                p[i][j] = s <= t ? s_t[t * DC_PITCH + s] * s_beta[half][s] : 0.f;
                most = fmaxf(most, fabsf(p[i][j]));
            }
        }
        most = dc_half_max(most, s_m, half);
        dc_scale(most, up, unit);
        if (ht == 0u) meta->f_t = unit;
#pragma unroll
        for (int i = 0; i < 4; ++i) { const uint32_t id = ht + i * 128u; put(p[i], up, id >> 3, id & 7u, rec); }
        dc_half_sync(half);
    }
}

// ---- the states through their chunks -------------------------------------------------------------------------------------------------------------
// A warp has 16 rows of a state as accumulators of m16n8k16 (64 registers), and what is computed for a row needs no other row, so warps share nothing but the chunk's operands in shared memory
// and meet once a chunk: S k and S q (operand A: the state's digits), R, D = T R (A: R's digits), the outputs (A: D's), the state (A: those of D times its decays). An accumulator's layout is that of
// an operand A, so that nothing is exchanged between lanes. The scale of a row's digits is its own.
// Chunk by chunk the operands come by bulk copies into one of two stages.
constexpr uint32_t DC_SPIN_LIMIT = 1u << 22;     // polls of a try_wait that is itself limited in time: far beyond any real wait

// the digits of x (rows g and g + 8 of a 16 x 16 step) as operand A
__device__ __forceinline__ void dc_operand(const float (&x0)[4], const float (&x1)[4], float up0, float up1, uint32_t (&hi)[4], uint32_t (&lo)[4]) {
    dc_digits(x0[0] * up0, x0[1] * up0, hi[0], lo[0]);
    dc_digits(x0[2] * up1, x0[3] * up1, hi[1], lo[1]);
    dc_digits(x1[0] * up0, x1[1] * up0, hi[2], lo[2]);
    dc_digits(x1[2] * up1, x1[3] * up1, hi[3], lo[3]);
}
template <int N>
__device__ __forceinline__ void dc_row_scale(const float (&x)[N][4], float (&up)[2], float (&unit)[2]) {
    float a = 0.f, b = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) { a = fmaxf(a, fmaxf(fabsf(x[i][0]), fabsf(x[i][1]))); b = fmaxf(b, fmaxf(fabsf(x[i][2]), fabsf(x[i][3]))); }
#pragma unroll
    for (int w = 1; w < 4; w <<= 1) { a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, w)); b = fmaxf(b, __shfl_xor_sync(0xffffffffu, b, w)); }
    dc_scale(a, up[0], unit[0]);
    dc_scale(b, up[1], unit[1]);
}

template <class T, int DIG, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, 1) k_delta_chunk(DeltaArgs A, uint32_t n_seqs, const uint8_t *ws, uint64_t slots) {
    pdl_prologue();
    constexpr uint32_t KEYS = dc_keys(DIG), STAGE = KEYS + DC_REC;
    extern __shared__ __align__(128) uint8_t sm[];
    __shared__ __align__(8) uint64_t s_full[2];
    __shared__ uint32_t s_seq;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, g = lane >> 2, c2 = (lane & 3u) * 2u;
    const uint32_t h = blockIdx.x / (8u / WARPS), j0 = (blockIdx.x % (8u / WARPS)) * (WARPS * 16u) + warp * 16u, kh = h / (A.rank / A.groups);
    // long sequences first: the block's sequence is the blockIdx.y-th longest (of many, they are taken as they come)
    uint32_t b = blockIdx.y + A.first_seq;
    if (n_seqs > 1u && n_seqs <= 1024u) {
        for (uint32_t i = tid; i < n_seqs; i += WARPS * 32u) {
            const int64_t mine = (int64_t)A.cu[i + 1u] - A.cu[i];
            uint32_t before = 0u;
            for (uint32_t j = 0; j < n_seqs; ++j) { const int64_t other = (int64_t)A.cu[j + 1u] - A.cu[j]; before += other > mine || (other == mine && j < i); }
            if (before == blockIdx.y) s_seq = i;
        }
        __syncthreads();
        b = s_seq;
    }
    const int32_t lo = A.cu[b], hi = A.cu[b + 1u];
    if (lo < 0 || hi < lo || (uint32_t)hi > A.n_tokens) { if (A.status && tid == 0u) A.status[ST_SEQ_BOUNDS] = 1u; return; }
    const int32_t state_slot = delta_slot(A.slots, A.n_slots, b, A.status);
    if (state_slot < 0 || lo == hi) return;
    const uint32_t len = (uint32_t)(hi - lo), chunks = (len + DC_T - 1u) / DC_T;
    const uint64_t slot0 = (uint64_t)(lo / DC_T) + b;
    const uint8_t *const keys = ws + (slot0 * A.groups + kh) * KEYS, *const recs = ws + slots * A.groups * KEYS + (slot0 * A.rank + h) * DC_REC;
    if (tid == 0u) {
        for (int i = 0; i < 2; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" :: "r"(dc_smem(&s_full[i])));
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    auto fetch = [&](uint32_t c) {               // by thread 0
        const uint32_t bar = dc_smem(&s_full[c & 1u]), dst = dc_smem(sm) + (c & 1u) * STAGE;
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" :: "r"(bar), "r"(STAGE) : "memory");
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                     :: "r"(dst), "l"(keys + (uint64_t)c * A.groups * KEYS), "r"(KEYS), "r"(bar) : "memory");
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                     :: "r"(dst + KEYS), "l"(recs + (uint64_t)c * A.rank * DC_REC), "r"(DC_REC), "r"(bar) : "memory");
    };
    auto wait = [&](uint32_t c) {
        uint32_t done = 0;
        for (uint32_t i = 0; i < DC_SPIN_LIMIT && !done; ++i)
            asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
                         : "=r"(done) : "r"(dc_smem(&s_full[c & 1u])), "r"((c >> 1) & 1u) : "memory");
        return done != 0u;
    };
    if (tid == 0u) fetch(0u);
    float *const state = A.state + (((uint64_t)(uint32_t)state_slot * A.rank + h) * DC_S + j0 + g) * DC_S + c2;      // rows g and g + 8, columns 8 i + c2, + 1
    float s[16][4];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float2 x = *reinterpret_cast<const float2 *>(state + i * 8), y = *reinterpret_cast<const float2 *>(state + 8 * DC_S + i * 8);
        s[i][0] = x.x; s[i][1] = x.y; s[i][2] = y.x; s[i][3] = y.y;
    }
    bool nan0 = false, nan1 = false;             // rows g, g + 8 are no numbers any more
    {
        bool f0 = true, f1 = true;
#pragma unroll
        for (int i = 0; i < 16; ++i) { f0 &= fabsf(s[i][0]) < INFINITY && fabsf(s[i][1]) < INFINITY; f1 &= fabsf(s[i][2]) < INFINITY && fabsf(s[i][3]) < INFINITY; }
        const uint32_t m0 = __ballot_sync(0xffffffffu, !f0), m1 = __ballot_sync(0xffffffffu, !f1), quad = 0xfu << (lane & 28u);
        nan0 = m0 & quad; nan1 = m1 & quad;
    }
    const T *const v = reinterpret_cast<const T *>(A.v) + (uint64_t)h * DC_S + j0 + g;
    T *const out = reinterpret_cast<T *>(A.out) + (uint64_t)h * DC_S + j0 + g;
    const uint32_t br = (lane & 7u) + (lane >> 4) * 8u, bc = (lane >> 3) & 1u;       // operand B from rows [n][k]: 16 rows, two pieces
    const uint32_t tr = (lane & 7u) + ((lane >> 3) & 1u) * 8u, tc = lane >> 4;       // from rows [k][n]: 16 rows, two pieces
    bool failed = false;
#pragma unroll 1
    for (uint32_t c = 0; c < chunks; ++c) {
        __syncthreads();                         // the other stage's chunk has been worked on
        if (tid == 0u && c + 1u < chunks) fetch(c + 1u);
        const uint32_t t0 = (uint32_t)lo + c * DC_T, n = min((uint32_t)DC_T, (uint32_t)hi - t0);
        // the chunk's values: token 8 i + c2 (+ 1), rows g and g + 8
        float r[8][4];
#pragma unroll
        for (uint32_t i = 0; i < 8u; ++i)
#pragma unroll
            for (uint32_t e = 0; e < 2u; ++e) {
                const uint32_t t = i * 8u + c2 + e;
                r[i][e] = r[i][e + 2] = 0.f;
                if (t < n) { r[i][e] = to_f32(v[(uint64_t)(t0 + t) * A.v_stride]); r[i][e + 2] = to_f32(v[(uint64_t)(t0 + t) * A.v_stride + 8u]); }
            }
        uint8_t *const st = sm + (c & 1u) * STAGE;
        const uint32_t k_at = dc_smem(st), q_at = k_at + DIG * DC_TILE, t_at = k_at + KEYS, p_at = t_at + 2u * DC_SQ;
        const DcMeta &M = *reinterpret_cast<const DcMeta *>(st + KEYS + 4u * DC_SQ);
        if (!wait(c)) { failed = true; break; }
        // the first token from which a row is no number (64: none)
        uint32_t from0 = nan0 ? 0u : M.nan_from, from1 = nan1 ? 0u : M.nan_from;
        {
            bool fine = true;
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) fine &= fabsf(r[i][e]) < INFINITY;
            if (!__all_sync(0xffffffffu, fine)) {
#pragma unroll
                for (uint32_t i = 0; i < 8u; ++i)
#pragma unroll
                    for (uint32_t e = 0; e < 4u; ++e)
                        if (!(fabsf(r[i][e]) < INFINITY)) {
                            uint32_t &from = e < 2u ? from0 : from1;
                            from = min(from, i * 8u + c2 + (e & 1u));
                            r[i][e] = 0.f;
                        }
#pragma unroll
                for (int w = 1; w < 4; w <<= 1) { from0 = min(from0, __shfl_xor_sync(0xffffffffu, from0, w)); from1 = min(from1, __shfl_xor_sync(0xffffffffu, from1, w)); }
            }
            if (nan0)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i][0] = s[i][1] = 0.f;
            if (nan1)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i][2] = s[i][3] = 0.f;
        }
        float up[2], unit[2], ks[8][4], o[8][4];
        dc_row_scale(s, up, unit);
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) ks[i][e] = o[i][e] = 0.f;
#pragma unroll
        for (uint32_t k = 0; k < 8u; ++k) {      // 16 columns of the state
            uint32_t ah[4], al[4];
            dc_operand(s[2 * k], s[2 * k + 1], up[0], up[1], ah, al);
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i) {  // 16 tokens
                uint32_t x[4], y[4];
                dc_ldsm(x, k_at + dc_tile_at(i * 16u + br, 2u * k + bc));
                dc_ldsm(y, q_at + dc_tile_at(i * 16u + br, 2u * k + bc));
                dc_mma(ks[2 * i], ah, x[0], x[1]); dc_mma(ks[2 * i + 1], ah, x[2], x[3]);
                dc_mma(o[2 * i], ah, y[0], y[1]); dc_mma(o[2 * i + 1], ah, y[2], y[3]);
                dc_mma(ks[2 * i], al, x[0], x[1]); dc_mma(ks[2 * i + 1], al, x[2], x[3]);
                dc_mma(o[2 * i], al, y[0], y[1]); dc_mma(o[2 * i + 1], al, y[2], y[3]);
                if (DIG == 2) {
                    dc_ldsm(x, k_at + DC_TILE + dc_tile_at(i * 16u + br, 2u * k + bc));
                    dc_ldsm(y, q_at + DC_TILE + dc_tile_at(i * 16u + br, 2u * k + bc));
                    dc_mma(ks[2 * i], ah, x[0], x[1]); dc_mma(ks[2 * i + 1], ah, x[2], x[3]);
                    dc_mma(o[2 * i], ah, y[0], y[1]); dc_mma(o[2 * i + 1], ah, y[2], y[3]);
                }
            }
        }
        {   // R, and the state's part of the outputs
            const float fk0 = unit[0] * M.f_k, fk1 = unit[1] * M.f_k, fq0 = unit[0] * M.f_q, fq1 = unit[1] * M.f_q;
#pragma unroll
            for (uint32_t i = 0; i < 8u; ++i)
#pragma unroll
                for (uint32_t e = 0; e < 2u; ++e) {
                    const float dec = M.dec[i * 8u + c2 + e];
                    r[i][e] = fmaf(-dec, ks[i][e] * fk0, r[i][e]); r[i][e + 2] = fmaf(-dec, ks[i][e + 2] * fk1, r[i][e + 2]);
                    o[i][e] *= dec * fq0; o[i][e + 2] *= dec * fq1;
                }
        }
        float d[8][4];
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) d[i][e] = 0.f;
        // x += (digits of y) * (the lower triangle at `at`)
        auto triangle = [&](float (&x)[8][4], const float (&y)[8][4], uint32_t at) {
#pragma unroll
            for (uint32_t k = 0; k < 4u; ++k) {
                uint32_t ah[4], al[4];
                dc_operand(y[2 * k], y[2 * k + 1], up[0], up[1], ah, al);
#pragma unroll
                for (uint32_t i = k; i < 4u; ++i) {
                    uint32_t z[4];
                    dc_ldsm(z, at + dc_sq_at(i * 16u + br, 2u * k + bc));
                    dc_mma(x[2 * i], ah, z[0], z[1]); dc_mma(x[2 * i + 1], ah, z[2], z[3]);
                    dc_mma(x[2 * i], al, z[0], z[1]); dc_mma(x[2 * i + 1], al, z[2], z[3]);
                    dc_ldsm(z, at + DC_SQ + dc_sq_at(i * 16u + br, 2u * k + bc));
                    dc_mma(x[2 * i], ah, z[0], z[1]); dc_mma(x[2 * i + 1], ah, z[2], z[3]);
                }
            }
        };
        dc_row_scale(r, up, unit);
        triangle(d, r, t_at);
#pragma unroll
        for (int i = 0; i < 8; ++i) { d[i][0] *= unit[0] * M.f_t; d[i][1] *= unit[0] * M.f_t; d[i][2] *= unit[1] * M.f_t; d[i][3] *= unit[1] * M.f_t; }
        dc_row_scale(d, up, unit);
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) r[i][e] = 0.f;
        triangle(r, d, p_at);
        {
            const float f0 = unit[0] * M.f_p, f1 = unit[1] * M.f_p;
            const bool numbers = from0 >= (uint32_t)DC_T && from1 >= (uint32_t)DC_T && !(M.bad_q[0] | M.bad_q[1]);
#pragma unroll
            for (uint32_t i = 0; i < 8u; ++i)
#pragma unroll
                for (uint32_t e = 0; e < 2u; ++e) {
                    const uint32_t t = i * 8u + c2 + e;
                    float y0 = A.scale * fmaf(r[i][e], f0, o[i][e]), y1 = A.scale * fmaf(r[i][e + 2], f1, o[i][e + 2]);
                    if (!numbers) {
                        const bool bad = (M.bad_q[t >> 5] >> (t & 31u)) & 1u;
                        if (bad || t >= from0) y0 = NAN;
                        if (bad || t >= from1) y1 = NAN;
                    }
                    if (t < n) {
                        T *const p = out + (uint64_t)(t0 + t) * A.rank * DC_S;
                        p[0] = from_f32<T>(y0); p[8] = from_f32<T>(y1);
                    }
                }
        }
        // the state
#pragma unroll
        for (uint32_t i = 0; i < 8u; ++i)
#pragma unroll
            for (uint32_t e = 0; e < 2u; ++e) { const float w = M.kdec[i * 8u + c2 + e]; d[i][e] *= w; d[i][e + 2] *= w; }
        dc_row_scale(d, up, unit);
        uint32_t dh[4][4], dl[4][4];
#pragma unroll
        for (int k = 0; k < 4; ++k) dc_operand(d[2 * k], d[2 * k + 1], up[0], up[1], dh[k], dl[k]);
        const float f0 = unit[0] * M.f_k, f1 = unit[1] * M.f_k, last = M.last;
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {      // 32 columns
            float x[4][4];
#pragma unroll
            for (int a = 0; a < 4; ++a)
#pragma unroll
                for (int e = 0; e < 4; ++e) x[a][e] = 0.f;
#pragma unroll
            for (uint32_t k = 0; k < 4u; ++k)
#pragma unroll
                for (uint32_t a = 0; a < 2u; ++a) {
                    uint32_t y[4];
                    dc_ldsm_t(y, k_at + dc_tile_at(k * 16u + tr, i * 4u + a * 2u + tc));
                    dc_mma(x[2 * a], dh[k], y[0], y[1]); dc_mma(x[2 * a + 1], dh[k], y[2], y[3]);
                    dc_mma(x[2 * a], dl[k], y[0], y[1]); dc_mma(x[2 * a + 1], dl[k], y[2], y[3]);
                    if (DIG == 2) {
                        dc_ldsm_t(y, k_at + DC_TILE + dc_tile_at(k * 16u + tr, i * 4u + a * 2u + tc));
                        dc_mma(x[2 * a], dh[k], y[0], y[1]); dc_mma(x[2 * a + 1], dh[k], y[2], y[3]);
                    }
                }
#pragma unroll
            for (uint32_t a = 0; a < 4u; ++a) {
                float (&y)[4] = s[4 * i + a];
                y[0] = fmaf(x[a][0], f0, y[0] * last); y[1] = fmaf(x[a][1], f0, y[1] * last);
                y[2] = fmaf(x[a][2], f1, y[2] * last); y[3] = fmaf(x[a][3], f1, y[3] * last);
            }
        }
        nan0 = from0 < (uint32_t)DC_T; nan1 = from1 < (uint32_t)DC_T;
    }
    if (failed) {                                // a copy never came: the next one is waited for, nothing more is written
        if (A.status && lane == 0u) A.status[ST_TIMEOUT] = 1u;
        for (uint32_t c = 0; c < chunks; ++c) if (!wait(c)) break;
        return;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        *reinterpret_cast<float2 *>(state + i * 8) = nan0 ? make_float2(NAN, NAN) : make_float2(s[i][0], s[i][1]);
        *reinterpret_cast<float2 *>(state + 8 * DC_S + i * 8) = nan1 ? make_float2(NAN, NAN) : make_float2(s[i][2], s[i][3]);
    }
}

uint64_t delta_chunk_workspace(uint32_t type, uint32_t groups, uint32_t rank, uint32_t n_tokens, uint32_t n_seqs) {
    return dc_slots(n_tokens, n_seqs) * ((uint64_t)groups * dc_keys(type == VT_F32 ? 2 : 1) + (uint64_t)rank * DC_REC);
}

template <class T, int DIG, int WARPS> static int launch_chunk(DeltaArgs A, uint32_t n_seqs, const uint8_t *ws, uint64_t slots, cudaStream_t s) {
    constexpr size_t smem = 2u * (dc_keys(DIG) + DC_REC);
    static std::atomic<uint64_t> set{0};
    if (!raise_smem_limit(reinterpret_cast<const void *>(k_delta_chunk<T, DIG, WARPS>), smem, set)) return 0;
    for (uint32_t b = 0; b < n_seqs; b += 65535u) {
        A.first_seq = b;
        RC_LAUNCH((k_delta_chunk<T, DIG, WARPS>), dim3(A.rank * (8u / WARPS), n_seqs - b < 65535u ? n_seqs - b : 65535u), WARPS * 32, smem, s, A, n_seqs, ws, slots);
        RC_LAUNCHED();
    }
    return 1;
}
template <class T, int DIG> static int launch_chunks(const DeltaArgs &A, uint32_t n_seqs, uint8_t *ws, cudaStream_t s) {
    const uint64_t slots = dc_slots(A.n_tokens, n_seqs);
    constexpr uint32_t region = 4u * DC_MAT > dc_keys(DIG) ? 4u * DC_MAT : dc_keys(DIG);
    constexpr size_t smem = 2u * DC_MAT + region;
    static std::atomic<uint64_t> set{0};
    if (!raise_smem_limit(reinterpret_cast<const void *>(k_delta_prep<T, DIG>), smem, set)) return 0;
    RC_REQUIRE(slots <= 0x7fffffffu && A.groups <= 65535u, "delta rule: too many chunks");
    prof_begin("delta_prep", s);
    RC_LAUNCH((k_delta_prep<T, DIG>), dim3((uint32_t)slots, A.groups), 256, smem, s, A, n_seqs, ws, slots);
    RC_LAUNCHED();
    prof_end(s);
    prof_begin("delta_chunk", s);
    const uint64_t heads = (uint64_t)n_seqs * A.rank;
    const int ok = heads * 4u <= sm_count() ? launch_chunk<T, DIG, 2>(A, n_seqs, ws, slots, s) : launch_chunk<T, DIG, 8>(A, n_seqs, ws, slots, s);
    prof_end(s);
    return ok;
}

int launch_delta_chunks(const DeltaArgs &A, uint32_t type, uint32_t n_seqs, uint8_t *ws, cudaStream_t s) {
    return type == VT_F32 ? launch_chunks<float, 2>(A, n_seqs, ws, s) : type == VT_F16 ? launch_chunks<__half, 1>(A, n_seqs, ws, s) : launch_chunks<__nv_bfloat16, 1>(A, n_seqs, ws, s);
}

}  // namespace rc
