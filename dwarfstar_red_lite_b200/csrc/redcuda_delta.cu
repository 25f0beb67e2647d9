// The gated delta rule by itself, for a batch of sequences with states in slots (the recurrence of native/redlite_native_engine_cpu.c:198-216):
//     S <- exp(g) S;   d = beta (v - S k);   S <- S + d k^T;   out = scale S q
//
//   k_delta_scan  one token of each sequence (STEP), or whole sequences laid end to end, a token at a time
//   k_delta_prep, k_delta_chunk (redcuda_delta_chunk.cu)  whole sequences in chunks on the tensor cores
#include "redcuda_delta.cuh"
#include "redcuda_stage.cuh"
#include "../../include/redcuda.h"

#include <math.h>

namespace rc {

// Lanes of a row: S / E of them with E columns each, in pieces of four columns that lie 4 S / E apart, so that a quarter warp reads 128 bytes in a row.
template <int S> struct DeltaLanes {
    static constexpr int E = S == 256 ? 8 : 4, LPR = S / E, RPW = 32 / LPR;      // a warp reads RPW rows at once
};

// The sums of N values over the LPR lanes of a row, N a power of two and at most LPR: value i ends in lane i of each run of N lanes ... every exchange
// halves the values that a lane carries.
template <int N, int LPR>
__device__ __forceinline__ float row_sums(float (&x)[N], uint32_t p) {
    int n = N;
#pragma unroll
    for (int w = LPR / 2; w; w >>= 1) {
        if (n > 1) {
            n /= 2;
            const bool hi = p & (uint32_t)w;
#pragma unroll
            for (int i = 0; i < N / 2; ++i)
                if (i < n) {
                    const float keep = hi ? x[n + i] : x[i], send = hi ? x[i] : x[n + i];
                    x[i] = keep + __shfl_xor_sync(0xffffffffu, send, w);
                }
        } else {
            x[0] += __shfl_xor_sync(0xffffffffu, x[0], w);
        }
    }
    return x[0];
}

// A block has ROWS rows of one head's state, in registers from the first token to the last. For a row m of the state before a token
//     S k = a (m . k),  S q = a (m . q) + d (k . q),  a = exp(g),
// so that both products of a row are summed over its lanes in one exchange.
// STEP: one token per sequence, token b; otherwise the tokens cu[b] .. cu[b + 1] - 1.
// What bounds the step is the state, read once and written once: 96 sequences of 32 heads x 128 x 128 (403 MB) take 62 us, 6.5 TB/s; one sequence 2.3 us, a launch. Blocks of 32 rows, so that one
// sequence is 128 of them. What bounds the scan is the chain of a token (two products, an exchange, the correction): some 0.29 us a token for F32 rows, 0.42 for 16 bits.
template <class T, int S, bool STEP>
__global__ void __launch_bounds__(DELTA_WARPS * 32) k_delta_scan(DeltaArgs A) {
    pdl_prologue();
    using L = DeltaLanes<S>;
    constexpr int E = L::E, LPR = L::LPR, RPW = L::RPW, R = DELTA_ROWS / (DELTA_WARPS * RPW);        // R rows a lane
    static_assert(S % DELTA_ROWS == 0 && R >= 1 && 2 * R <= LPR, "rows of a block");
    constexpr int SPLIT = S / DELTA_ROWS;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, p = lane % LPR, r = lane / LPR;
    const uint32_t h = blockIdx.x / SPLIT, j0 = (blockIdx.x % SPLIT) * DELTA_ROWS + warp * (RPW * R), b = blockIdx.y + A.first_seq, kh = h / (A.rank / A.groups);
    int32_t t0, t1;
    if (STEP) { t0 = (int32_t)b; t1 = t0 + 1; } else { t0 = A.cu[b]; t1 = A.cu[b + 1u]; }
    if (!STEP && (t0 < 0 || t1 < t0 || (uint32_t)t1 > A.n_tokens)) { if (A.status && tid == 0u) A.status[ST_SEQ_BOUNDS] = 1u; return; }
    const int32_t slot = delta_slot(A.slots, A.n_slots, b, A.status);
    if (slot < 0 || t0 == t1) return;
    float *state = A.state + (((uint64_t)(uint32_t)slot * A.rank + h) * S + j0) * S;
    auto col = [&](int i) { return (uint32_t)((i / 4) * 4 * LPR) + p * 4u; };      // first of the columns i .. i + 3
    float m[R][E];
#pragma unroll
    for (int a = 0; a < R; ++a)
#pragma unroll
        for (int i = 0; i < E; i += 4) *reinterpret_cast<float4 *>(&m[a][i]) = *reinterpret_cast<const float4 *>(state + (uint64_t)(a * RPW + r) * S + col(i));
    const T *q = reinterpret_cast<const T *>(A.q) + (uint64_t)(uint32_t)t0 * A.q_stride + (uint64_t)kh * S;
    const T *k = reinterpret_cast<const T *>(A.k) + (uint64_t)(uint32_t)t0 * A.k_stride + (uint64_t)kh * S;
    const T *v = reinterpret_cast<const T *>(A.v) + (uint64_t)(uint32_t)t0 * A.v_stride + (uint64_t)h * S + j0;
    T *out = reinterpret_cast<T *>(A.out) + ((uint64_t)(uint32_t)t0 * A.rank + h) * S + j0;
    const float *gate = A.gate + (uint64_t)(uint32_t)t0 * A.rank + h, *beta = A.beta + (uint64_t)(uint32_t)t0 * A.rank + h;
    // after row_sums lane p of a row holds value which / (LPR / (2 R)): S k of row `mine` in the lower half, S q in the upper
    constexpr int STEPS = LPR / (2 * R);
    const uint32_t val = p / STEPS, mine = val % R;
    const bool holds_q = val >= (uint32_t)R;
    float kk[E], qq[E], vv = 0.f, gg = 0.f, bb = 0.f;
    auto load = [&](uint32_t t) {
#pragma unroll
        for (int i = 0; i < E; i += 4) {
            load_vals<4>(k + (uint64_t)t * A.k_stride + col(i), *reinterpret_cast<float (*)[4]>(&kk[i]));
            load_vals<4>(q + (uint64_t)t * A.q_stride + col(i), *reinterpret_cast<float (*)[4]>(&qq[i]));
        }
        vv = to_f32(v[(uint64_t)t * A.v_stride + mine * RPW + r]);
        gg = gate[(uint64_t)t * A.rank]; bb = beta[(uint64_t)t * A.rank];
    };
    load(0u);
    const uint32_t n = (uint32_t)(t1 - t0);
    for (uint32_t t = 0; t < n; ++t) {
        float kc[E], x[2 * R], kq = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) { kc[i] = kk[i]; kq += kk[i] * qq[i]; }
#pragma unroll
        for (int a = 0; a < R; ++a) {
            x[a] = m[a][0] * kc[0]; x[R + a] = m[a][0] * qq[0];
#pragma unroll
            for (int i = 1; i < E; ++i) { x[a] += m[a][i] * kc[i]; x[R + a] += m[a][i] * qq[i]; }
        }
        const float dec = expf(gg), bt = bb, vt = vv;
        if (!STEP && t + 1u < n) load(t + 1u);
#pragma unroll
        for (int w = LPR / 2; w; w >>= 1) kq += __shfl_xor_sync(0xffffffffu, kq, w);
        const float s = dec * row_sums<2 * R, LPR>(x, p);
        const float d_mine = (vt - s) * bt;       // in the lanes that hold S k
        float d[R];
#pragma unroll
        for (int a = 0; a < R; ++a) d[a] = __shfl_sync(0xffffffffu, d_mine, (int)(lane - p) + a * STEPS);
#pragma unroll
        for (int a = 0; a < R; ++a)
#pragma unroll
            for (int i = 0; i < E; ++i) m[a][i] = fmaf(d[a], kc[i], m[a][i] * dec);
        const float dq = __shfl_sync(0xffffffffu, d_mine, (int)(lane - p) + (int)mine * STEPS);
        if (holds_q && p % STEPS == 0u) out[(uint64_t)t * A.rank * S + mine * RPW + r] = from_f32<T>((s + dq * kq) * A.scale);
    }
#pragma unroll
    for (int a = 0; a < R; ++a)
#pragma unroll
        for (int i = 0; i < E; i += 4) *reinterpret_cast<float4 *>(state + (uint64_t)(a * RPW + r) * S + col(i)) = *reinterpret_cast<const float4 *>(&m[a][i]);
}

template <class T, int S, bool STEP> static int launch_scan(DeltaArgs A, uint32_t n_seqs, cudaStream_t s) {
    for (uint32_t b = 0; b < n_seqs; b += 65535u) {
        A.first_seq = b;
        RC_LAUNCH((k_delta_scan<T, S, STEP>), dim3(A.rank * (S / DELTA_ROWS), n_seqs - b < 65535u ? n_seqs - b : 65535u), DELTA_WARPS * 32, 0, s, A);
        RC_LAUNCHED();
    }
    return 1;
}
template <class T, bool STEP> static int launch_scan_s(const DeltaArgs &A, uint32_t S, uint32_t n_seqs, cudaStream_t s) {
    return S == 256u ? launch_scan<T, 256, STEP>(A, n_seqs, s) : S == 128u ? launch_scan<T, 128, STEP>(A, n_seqs, s) : S == 64u ? launch_scan<T, 64, STEP>(A, n_seqs, s) : launch_scan<T, 32, STEP>(A, n_seqs, s);
}
template <bool STEP> static int launch_scan_t(const DeltaArgs &A, uint32_t type, uint32_t S, uint32_t n_seqs, cudaStream_t s) {
    return type == VT_F32 ? launch_scan_s<float, STEP>(A, S, n_seqs, s) : type == VT_F16 ? launch_scan_s<__half, STEP>(A, S, n_seqs, s) : launch_scan_s<__nv_bfloat16, STEP>(A, S, n_seqs, s);
}

// In chunks on the tensor cores, or a token at a time: a chunk costs nearly the same whatever it holds, and the first one of a call 20 us. us with 32 heads, a token at a time -> in chunks, F32 (BF16):
// 1 sequence of 32 tokens 12 -> 24 (16 -> 20), of 64 21 -> 26 (30 -> 21), of 128 39 -> 30 (58 -> 26); 4 of 32 30 -> 33 (35 -> 26); 16 of 16 42 -> 71 (49 -> 58), of 32 79 -> 75 (91 -> 61);
// 64 of 16 172 -> 244 (198 -> 221), of 32 316 -> 258 (371 -> 227). The crossing lies at some 25 tokens a sequence and 50 more for F32, 18 and 20 for 16 bits; one rule between them.
static bool delta_in_chunks(const redcuda_delta_dims *d, uint32_t n_tokens, uint32_t n_seqs) { return d->d_state == 128u && n_tokens >= 24u * (uint64_t)n_seqs + 32u; }

// What a call's arguments have to be; fills the strides. rows: tokens of q, k, v and out
static int delta_check(const redcuda_delta_dims *d, const char *who, uint32_t rows, uint32_t n_seqs, uint32_t n_slots, DeltaArgs &A) {
    RC_REQUIRE(d, "%s: null dimensions", who);
    const uint32_t size = val_size(d->type);
    RC_REQUIRE(size, "%s: rows of type %u (F32, F16 or BF16 are served)", who, d->type);
    RC_REQUIRE(d->d_state == 32u || d->d_state == 64u || d->d_state == 128u || d->d_state == 256u, "%s: states of %u (32, 64, 128 or 256 are served)", who, d->d_state);
    RC_REQUIRE(d->n_group && d->dt_rank && d->dt_rank % d->n_group == 0u && d->dt_rank <= 65535u, "%s: %u value heads over %u key heads", who, d->dt_rank, d->n_group);
    RC_REQUIRE(rows < 0x7fffffffu && n_seqs < 0x7fffffffu, "%s: too many rows", who);
    RC_REQUIRE(n_slots && n_slots <= 0x7fffffffu, "%s: no states", who);
    const uint64_t key = (uint64_t)d->n_group * d->d_state, val = (uint64_t)d->dt_rank * d->d_state;
    A.q_stride = d->q_stride ? d->q_stride : key;
    A.k_stride = d->k_stride ? d->k_stride : key;
    A.v_stride = d->v_stride ? d->v_stride : val;
    RC_REQUIRE(A.q_stride >= key && A.k_stride >= key && A.v_stride >= val && A.q_stride * size % 16u == 0u && A.k_stride * size % 16u == 0u && A.v_stride * size % 16u == 0u &&
               A.q_stride < (1ull << 32) && A.k_stride < (1ull << 32) && A.v_stride < (1ull << 32), "%s: row strides (multiples of 16 bytes, at least a row)", who);
    RC_REQUIRE(!(d->scale != d->scale), "%s: scale is not a number", who);
    A.scale = d->scale == 0.f ? (float)(1.0 / sqrt((double)d->d_state)) : d->scale;
    A.n_tokens = rows; A.n_slots = n_slots; A.groups = d->n_group; A.rank = d->dt_rank;
    return 1;
}
static int delta_pointers(const redcuda_delta_dims *d, const char *who, uint32_t rows, uint32_t n_seqs, uint32_t n_slots, const DeltaArgs &A) {
    RC_REQUIRE(A.q && A.k && A.v && A.gate && A.beta && A.state && A.out, "%s: null argument", who);
    RC_REQUIRE(aligned16(A.q) && aligned16(A.k) && aligned16(A.v) && aligned16(A.state) && aligned16(A.out), "%s: a pointer is not 16-byte aligned", who);
    RC_REQUIRE(aligned4(A.gate) && aligned4(A.beta) && aligned4(A.slots) && aligned4(A.cu), "%s: gates, betas or whole numbers are not 4-byte aligned", who);
    const uint32_t size = val_size(d->type);
    const uint64_t key = (uint64_t)d->n_group * d->d_state, val = (uint64_t)d->dt_rank * d->d_state, ob = (uint64_t)rows * val * size, sb = (uint64_t)n_slots * val * d->d_state * 4u;
    const void *in[7] = {A.q, A.k, A.v, A.gate, A.beta, A.cu, A.slots};
    const uint64_t bytes[7] = {span_bytes(rows, A.q_stride, key, size), span_bytes(rows, A.k_stride, key, size), span_bytes(rows, A.v_stride, val, size), (uint64_t)rows * d->dt_rank * 4u,
                               (uint64_t)rows * d->dt_rank * 4u, (n_seqs + 1ull) * 4u, (uint64_t)n_seqs * 4u};
    for (int i = 0; i < 7; ++i) RC_REQUIRE(!overlap(A.out, ob, in[i], bytes[i]) && !overlap(A.state, sb, in[i], bytes[i]), "%s: the output or the states lie inside the inputs", who);
    RC_REQUIRE(!overlap(A.out, ob, A.state, sb), "%s: the output lies inside the states", who);
    return 1;
}

}  // namespace rc

using namespace rc;

extern "C" {

int redcuda_delta_step_device(const redcuda_delta_dims *d, uint32_t n_seqs, const int32_t *slots_dev, uint32_t n_slots, const void *q_dev, const void *k_dev,
                              const void *v_dev, const float *gate_dev, const float *beta_dev, float *state_dev, void *out_dev, void *stream) {
    DeltaArgs A{};
    if (!delta_check(d, "delta step", n_seqs, n_seqs, n_slots, A)) return 0;
    A.q = q_dev; A.k = k_dev; A.v = v_dev; A.gate = gate_dev; A.beta = beta_dev; A.state = state_dev; A.out = out_dev; A.slots = slots_dev;
    RC_REQUIRE(n_seqs, "delta step: no sequences");
    RC_REQUIRE(slots_dev || n_seqs <= n_slots, "delta step: %u sequences for %u states", n_seqs, n_slots);
    if (!delta_pointers(d, "delta step", n_seqs, n_seqs, n_slots, A) || !require_device()) return 0;
    A.status = status_words();
    cudaStream_t s = (cudaStream_t)stream;
    prof_begin("delta_step", s);
    const int ok = launch_scan_t<true>(A, d->type, d->d_state, n_seqs, s);
    prof_end(s);
    return ok;
}

uint64_t redcuda_delta_rule_workspace(const redcuda_delta_dims *d, uint32_t n_tokens, uint32_t n_seqs) {
    DeltaArgs A{};
    if (!delta_check(d, "delta rule", n_tokens, n_seqs, 1u, A)) return 0;
    return delta_in_chunks(d, n_tokens, n_seqs) ? delta_chunk_workspace(d->type, d->n_group, d->dt_rank, n_tokens, n_seqs) : 0u;
}

int redcuda_delta_rule_device(const redcuda_delta_dims *d, uint32_t n_tokens, uint32_t n_seqs, const int32_t *cu_seqlens_dev, const int32_t *slots_dev,
                              uint32_t n_slots, const void *q_dev, const void *k_dev, const void *v_dev, const float *gate_dev, const float *beta_dev,
                              float *state_dev, void *out_dev, void *workspace_dev, uint64_t workspace_bytes, void *stream) {
    DeltaArgs A{};
    if (!delta_check(d, "delta rule", n_tokens, n_seqs, n_slots, A)) return 0;
    A.q = q_dev; A.k = k_dev; A.v = v_dev; A.gate = gate_dev; A.beta = beta_dev; A.state = state_dev; A.out = out_dev; A.slots = slots_dev; A.cu = cu_seqlens_dev;
    RC_REQUIRE(n_seqs && cu_seqlens_dev, "delta rule: no sequences");
    RC_REQUIRE(slots_dev || n_seqs <= n_slots, "delta rule: %u sequences for %u states", n_seqs, n_slots);
    if (!delta_pointers(d, "delta rule", n_tokens, n_seqs, n_slots, A)) return 0;
    const uint64_t need = redcuda_delta_rule_workspace(d, n_tokens, n_seqs);
    RC_REQUIRE(!need || (workspace_dev && workspace_bytes >= need && aligned16(workspace_dev)), "delta rule: a 16-byte aligned workspace of %llu bytes is needed", (unsigned long long)need);
    if (need) {
        const uint32_t size = val_size(d->type);
        const uint64_t val = (uint64_t)d->dt_rank * d->d_state, rows = (uint64_t)n_tokens * d->dt_rank * 4u;
        RC_REQUIRE(!overlap(workspace_dev, need, out_dev, n_tokens * val * size) && !overlap(workspace_dev, need, state_dev, n_slots * val * d->d_state * 4u) &&
                   !overlap(workspace_dev, need, q_dev, span_bytes(n_tokens, A.q_stride, (uint64_t)d->n_group * d->d_state, size)) &&
                   !overlap(workspace_dev, need, k_dev, span_bytes(n_tokens, A.k_stride, (uint64_t)d->n_group * d->d_state, size)) &&
                   !overlap(workspace_dev, need, v_dev, span_bytes(n_tokens, A.v_stride, val, size)) && !overlap(workspace_dev, need, gate_dev, rows) && !overlap(workspace_dev, need, beta_dev, rows) &&
                   !overlap(workspace_dev, need, cu_seqlens_dev, (n_seqs + 1ull) * 4u) && !overlap(workspace_dev, need, slots_dev, (uint64_t)n_seqs * 4u),
                   "delta rule: the workspace overlaps rows, states, outputs, bounds or slots");
    }
    if (!require_device()) return 0;
    if (!n_tokens) return 1;
    A.status = status_words();
    cudaStream_t s = (cudaStream_t)stream;
    prof_begin("delta_rule", s);
    const int ok = delta_in_chunks(d, n_tokens, n_seqs) ? launch_delta_chunks(A, d->type, n_seqs, (uint8_t *)workspace_dev, s) : launch_scan_t<false>(A, d->type, d->d_state, n_seqs, s);
    prof_end(s);
    return ok;
}

int redcuda_delta_rule(const redcuda_delta_dims *d, uint32_t n_tokens, uint32_t n_seqs, const int32_t *cu_seqlens, const int32_t *slots, uint32_t n_slots,
                       const void *q, const void *k, const void *v, const float *gate, const float *beta, float *state, void *out) {
    DeltaArgs A{};
    if (!delta_check(d, "delta rule", n_tokens, n_seqs, n_slots, A)) return 0;
    RC_REQUIRE(q && k && v && gate && beta && state && out && cu_seqlens && n_seqs, "delta rule: null or empty argument");
    RC_REQUIRE(slots || n_seqs <= n_slots, "delta rule: %u sequences for %u states", n_seqs, n_slots);
    if (!require_device()) return 0;
    if (!n_tokens) return 1;
    const uint32_t size = val_size(d->type);
    const uint64_t key = (uint64_t)d->n_group * d->d_state, val = (uint64_t)d->dt_rank * d->d_state;
    const uint64_t qb = span_bytes(n_tokens, A.q_stride, key, size), kb = span_bytes(n_tokens, A.k_stride, key, size), vb = span_bytes(n_tokens, A.v_stride, val, size);
    const uint64_t gb = (uint64_t)n_tokens * d->dt_rank * 4u, sb = (uint64_t)n_slots * val * d->d_state * 4u, ob = (uint64_t)n_tokens * val * size, cb = (n_seqs + 1ull) * 4u, lb = n_seqs * 4ull;
    const uint64_t wb = redcuda_delta_rule_workspace(d, n_tokens, n_seqs);
    Stage st;
    if (!st.open(Stage::pad(qb) + Stage::pad(kb) + Stage::pad(vb) + 2u * Stage::pad(gb) + Stage::pad(sb) + Stage::pad(ob) + Stage::pad(cb) + Stage::pad(lb) + Stage::pad(wb))) return 0;
    uint8_t *dq = st.take(qb), *dk = st.take(kb), *dv = st.take(vb), *dg = st.take(gb), *db = st.take(gb), *ds = st.take(sb), *dout = st.take(ob), *dc = st.take(cb), *dl = st.take(lb), *dw = st.take(wb);
    if (!st.upload(dq, q, qb) || !st.upload(dk, k, kb) || !st.upload(dv, v, vb) || !st.upload(dg, gate, gb) || !st.upload(db, beta, gb) || !st.upload(ds, state, sb) || !st.upload(dc, cu_seqlens, cb) ||
        (slots && !st.upload(dl, slots, lb)) || !st.upload(dout, out, ob)) return 0;
    if (!redcuda_delta_rule_device(d, n_tokens, n_seqs, (const int32_t *)dc, slots ? (const int32_t *)dl : nullptr, n_slots, dq, dk, dv, (const float *)dg, (const float *)db, (float *)ds, dout, dw, wb,
                                   st.stream())) return 0;
    if (!st.download(state, ds, sb) || !st.download(out, dout, ob) || !st.finish()) return 0;
    return status_failed() ? 0 : 1;
}

}  // extern "C"
