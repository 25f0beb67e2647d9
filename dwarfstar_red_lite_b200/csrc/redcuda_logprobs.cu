// Log probability of a given token, entropy and the most likely alternatives of rows of logits, in one pass over them.
//
// A part of a row is summed up as m = max x, s = sum e^(x - m), u = sum e^(x - m) (x - m), and the n largest values; parts are joined by rescaling to
// the common m:  s' = s e^(m - m'),  u' = e^(m - m') (u + s (m - m')).  With these, lse = m + log s, entropy = log s - u / s.
// A cluster of blocks shares a row where there are few rows (LP_CLUSTER at most), so that the parts meet in shared memory and a call is one launch.
#include "redcuda_stage.cuh"
#include "redcuda_vals.cuh"
#include "../../include/redcuda.h"

#include <cooperative_groups.h>
#include <math.h>

namespace rc {

namespace cg = cooperative_groups;

constexpr int LP_WARPS = 8, LP_CLUSTER = 8, LP_TOP = (int)REDCUDA_MAX_ALTERNATIVES;

struct LogprobArgs {
    const void *x;
    uint64_t row_stride;
    const int32_t *tokens;
    float *logprob, *entropy, *top_lp;
    int32_t *top_ids;
    uint32_t *status;
    uint32_t vocab, top_n;
};

// The order of values, the lower index first among equal ones, as unsigned numbers: larger is earlier. Never 0 for a value.
__device__ __forceinline__ uint64_t lp_key(float x, uint32_t i) {
    const uint32_t b = __float_as_uint(x + 0.f);             // -0 is +0
    return (uint64_t)(b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u)) << 32 | (uint32_t)~i;
}
__device__ __forceinline__ float lp_value(uint64_t key) {
    const uint32_t o = (uint32_t)(key >> 32);
    return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
}

struct LpSums { float m, s, u; };
__device__ __forceinline__ LpSums lp_join(LpSums a, LpSums b) {
    LpSums r;
    r.m = fmaxf(a.m, b.m);
    const float z = r.m == -INFINITY ? 0.f : r.m, da = a.m - z, db = b.m - z, ea = expf(da), eb = expf(db);
    r.s = a.s * ea + b.s * eb;
    // a part that weighs nothing (an empty one, or one whose distance overflows) is not multiplied with it
    r.u = (ea > 0.f ? ea * (a.u + a.s * da) : 0.f) + (eb > 0.f ? eb * (b.u + b.s * db) : 0.f);
    return r;
}

template <class T>
__global__ void __launch_bounds__(LP_WARPS * 32) k_token_logprobs(LogprobArgs A) {
    pdl_prologue();
    constexpr int VEC = 16 / sizeof(T);
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t parts = cluster.num_blocks(), part = cluster.block_rank(), row = blockIdx.x / parts;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, n = A.top_n;
    __shared__ uint64_t s_keys[LP_WARPS * LP_TOP], s_best[LP_CLUSTER * LP_TOP];
    __shared__ LpSums s_sums[LP_WARPS > LP_CLUSTER ? LP_WARPS : LP_CLUSTER];
    const T *x = reinterpret_cast<const T *>(A.x) + (uint64_t)row * A.row_stride;
    // the row as up to VEC - 1 single values, whole 16-byte pieces, up to VEC - 1 single values
    const uint32_t head = min(A.vocab, (uint32_t)((16u - ((uintptr_t)x & 15u)) & 15u) / (uint32_t)sizeof(T)), pieces = (A.vocab - head) / VEC;
    const uint32_t per = (pieces + parts - 1u) / parts, p0 = min(pieces, part * per), p1 = min(pieces, p0 + per);

    LpSums S{-INFINITY, 0.f, 0.f};
    bool odd = false;                            // a NaN or +infinity
    uint64_t best = 0ull;                        // lane i: the i-th largest of what the warp has seen
    uint64_t least = 0ull;                       // the n-th
    auto sum = [&](float v) {
        odd |= !(v < INFINITY);
        if (v > S.m) {                           // never so for a NaN
            const float d = S.m - v, e = expf(d);
            S.u = e > 0.f ? e * (S.u + S.s * d) : 0.f;
            S.s *= e; S.m = v;
        }
        if (v > -INFINITY) {
            const float d = v - S.m, e = expf(d);
            S.s += e;
            S.u += e > 0.f ? e * d : 0.f;
        }
    };
    auto insert = [&](uint64_t key) {            // the same key in every lane
        const bool above = best >= key;
        const uint64_t up = __shfl_up_sync(0xffffffffu, best, 1);
        const bool above_up = lane == 0u || up >= key;
        best = above ? best : above_up ? key : up;
        least = __shfl_sync(0xffffffffu, best, (int)n - 1);
    };
    auto offer = [&](bool have, float v, uint32_t i) {        // by the whole warp
        if (n == 0u) return;
        const uint64_t key = have && v == v ? lp_key(v, i) : 0ull;
        for (uint32_t todo = __ballot_sync(0xffffffffu, key > least); todo; todo &= todo - 1u) {
            const uint64_t k = __shfl_sync(0xffffffffu, key, (int)__ffs((int)todo) - 1);
            if (k > least) insert(k);
        }
    };
    for (uint32_t p = p0 + warp * 32u; p < p1; p += LP_WARPS * 32u) {
        const bool have = p + lane < p1;
        float v[VEC] = {};
        if (have) load_vals<VEC>(x + head + (uint64_t)(p + lane) * VEC, v);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            if (have) sum(v[i]);
            offer(have, v[i], head + (p + lane) * VEC + i);
        }
    }
    if (part == 0u && warp == 0u) {              // the single values at both ends
        const uint32_t tail = head + pieces * VEC, ends = head + A.vocab - tail;
        const uint32_t i = lane < head ? lane : tail + lane - head;
        const bool have = lane < ends;
        const float v = have ? to_f32(x[i]) : 0.f;
        if (have) sum(v);
        offer(have, v, i);
    }
#pragma unroll
    for (int w = 16; w; w >>= 1) {
        LpSums o{__shfl_xor_sync(0xffffffffu, S.m, w), __shfl_xor_sync(0xffffffffu, S.s, w), __shfl_xor_sync(0xffffffffu, S.u, w)};
        S = lp_join(S, o);
    }
    if (__any_sync(0xffffffffu, odd)) S.s = NAN;
    if (lane == 0u) s_sums[warp] = S;
    if (lane < n) s_keys[warp * n + lane] = best;
    __syncthreads();
    // the n largest of the lists in s: every key finds its place by counting those above it (0: no value, no place)
    auto select = [&](const uint64_t *s, uint32_t count, uint64_t *to) {
        for (uint32_t i = tid; i < count; i += LP_WARPS * 32u) {
            const uint64_t key = s[i];
            uint32_t above = 0u;
            for (uint32_t j = 0; j < count; ++j) above += s[j] > key;
            if (key && above < n) to[above] = key;
        }
    };
    LpSums B = s_sums[0];
    for (int w = 1; w < LP_WARPS; ++w) B = lp_join(B, s_sums[w]);
    __syncthreads();
    cluster.sync();                              // the other blocks have begun: their shared memory may be written
    {
        uint64_t *to = cluster.map_shared_rank(s_best, 0) + part * n;
        for (uint32_t i = tid; i < n; i += LP_WARPS * 32u) to[i] = 0ull;
        __syncthreads();
        select(s_keys, LP_WARPS * n, to);
        if (tid == 0u) cluster.map_shared_rank(s_sums, 0)[part] = B;
    }
    cluster.sync();
    if (part != 0u) return;
    for (uint32_t i = tid; i < n; i += LP_WARPS * 32u) s_keys[i] = 0ull;
    __syncthreads();
    select(s_best, parts * n, s_keys);
    B = s_sums[0];
    for (uint32_t w = 1; w < parts; ++w) B = lp_join(B, s_sums[w]);
    __syncthreads();
    const float ls = logf(B.s);                              // nothing left: m = -infinity, s = 0
    const bool nan = !(B.s == B.s), none = !nan && B.m == -INFINITY;
    if (tid == 0u) {
        if (A.logprob) {
            const int32_t t = A.tokens[row];
            float lp = NAN;
            if (t >= 0 && (uint32_t)t < A.vocab) lp = nan ? NAN : none ? -INFINITY : (to_f32(x[t]) - B.m) - ls;
            else if (t != -1 && A.status) A.status[ST_TOKEN_RANGE] = 1u;
            A.logprob[row] = lp;
        }
        if (A.entropy) A.entropy[row] = nan ? NAN : none ? 0.f : fmaxf(ls - B.u / B.s, 0.f);
    }
    if (A.top_ids)
        for (uint32_t i = tid; i < n; i += LP_WARPS * 32u) {
            const uint64_t key = s_keys[i];
            A.top_ids[(uint64_t)row * n + i] = nan ? -1 : (int32_t)~(uint32_t)key;
            A.top_lp[(uint64_t)row * n + i] = nan ? NAN : none ? -INFINITY : (lp_value(key) - B.m) - ls;
        }
}

template <class T> static int launch_logprobs(const LogprobArgs &A, uint32_t rows, cudaStream_t s) {
    const uint32_t sms = sm_count();
    uint32_t parts = 1u;
    while (parts < (uint32_t)LP_CLUSTER && (uint64_t)rows * parts < 2u * sms && A.vocab / parts > 4096u) parts *= 2u;
    prof_begin("token_logprobs", s);
    for (uint64_t r = 0; r < rows; r += 1u << 24) {
        const uint32_t some = rows - r < 1u << 24 ? (uint32_t)(rows - r) : 1u << 24;
        LogprobArgs B = A;
        B.x = reinterpret_cast<const T *>(A.x) + r * A.row_stride;
        if (B.tokens) B.tokens += r;
        if (B.logprob) B.logprob += r;
        if (B.entropy) B.entropy += r;
        if (B.top_ids) { B.top_ids += r * A.top_n; B.top_lp += r * A.top_n; }
        RC_LAUNCH_CLUSTER(parts, (k_token_logprobs<T>), some * parts, LP_WARPS * 32, 0, s, B);
        RC_LAUNCHED();
    }
    prof_end(s);
    return 1;
}

static int logprobs_check(uint32_t type, uint32_t rows, uint32_t vocab, uint64_t &row_stride, const void *logits, const int32_t *tokens, uint32_t top_n, float *logprob, int32_t *top_ids, float *top_lp) {
    RC_REQUIRE(val_size(type), "token logprobs: logits of type %u (F32, F16 or BF16 are served)", type);
    RC_REQUIRE(logits && vocab && vocab < 0x7fffffffu && rows < 0x7fffffffu, "token logprobs: null or empty argument");
    if (!row_stride) row_stride = vocab;
    RC_REQUIRE(row_stride >= vocab && row_stride < (1ull << 32), "token logprobs: rows of %u values %llu apart", vocab, (unsigned long long)row_stride);
    RC_REQUIRE(top_n <= REDCUDA_MAX_ALTERNATIVES && top_n <= vocab, "token logprobs: %u alternatives of %u (at most %u)", top_n, vocab, REDCUDA_MAX_ALTERNATIVES);
    RC_REQUIRE((top_ids != nullptr) == (top_lp != nullptr) && (top_ids != nullptr) == (top_n != 0u), "token logprobs: alternatives need ids, log probabilities and a number of them");
    RC_REQUIRE(!logprob || tokens, "token logprobs: a log probability of no token");
    RC_REQUIRE((uintptr_t)logits % val_size(type) == 0u, "token logprobs: logits are not aligned to their type");
    return 1;
}

}  // namespace rc

using namespace rc;

extern "C" {

int redcuda_token_logprobs_device(uint32_t type, uint32_t rows, uint32_t vocab, uint64_t row_stride, const void *logits_dev, const int32_t *tokens_dev, uint32_t top_n,
                                  float *logprob_dev, float *entropy_dev, int32_t *top_ids_dev, float *top_logprobs_dev, void *stream) {
    if (!logprobs_check(type, rows, vocab, row_stride, logits_dev, tokens_dev, top_n, logprob_dev, top_ids_dev, top_logprobs_dev)) return 0;
    const uint64_t lb = span_bytes(rows, row_stride, vocab, val_size(type)), ob = (uint64_t)rows * 4u;
    RC_REQUIRE(!overlap(logits_dev, lb, logprob_dev, ob) && !overlap(logits_dev, lb, entropy_dev, ob) && !overlap(logits_dev, lb, top_ids_dev, ob * top_n) &&
               !overlap(logits_dev, lb, top_logprobs_dev, ob * top_n), "token logprobs: an output lies inside the logits");
    if (!require_device()) return 0;
    if (!rows) return 1;
    LogprobArgs A{logits_dev, row_stride, tokens_dev, logprob_dev, entropy_dev, top_logprobs_dev, top_ids_dev, status_words(), vocab, top_n};
    cudaStream_t s = (cudaStream_t)stream;
    return type == VT_F32 ? launch_logprobs<float>(A, rows, s) : type == VT_F16 ? launch_logprobs<__half>(A, rows, s) : launch_logprobs<__nv_bfloat16>(A, rows, s);
}

int redcuda_token_logprobs(uint32_t type, uint32_t rows, uint32_t vocab, uint64_t row_stride, const void *logits, const int32_t *tokens, uint32_t top_n,
                           float *logprob, float *entropy, int32_t *top_ids, float *top_logprobs) {
    if (!logprobs_check(type, rows, vocab, row_stride, logits, tokens, top_n, logprob, top_ids, top_logprobs) || !require_device()) return 0;
    if (!rows) return 1;
    const uint64_t lb = span_bytes(rows, row_stride, vocab, val_size(type)), rb = (uint64_t)rows * 4u, tb = rb * top_n;
    Stage st;
    if (!st.open(Stage::pad(lb) + 3u * Stage::pad(rb) + 2u * Stage::pad(tb))) return 0;
    uint8_t *x = st.take(lb);
    int32_t *t = st.take<int32_t>(rb);
    float *lp = st.take<float>(rb), *en = st.take<float>(rb);
    int32_t *ti = st.take<int32_t>(tb);
    float *tl = st.take<float>(tb);
    if (!st.upload(x, logits, lb) || (tokens && !st.upload(t, tokens, rb))) return 0;
    if (!redcuda_token_logprobs_device(type, rows, vocab, row_stride, x, tokens ? t : nullptr, top_n, logprob ? lp : nullptr, entropy ? en : nullptr, top_n ? ti : nullptr, top_n ? tl : nullptr, st.stream()))
        return 0;
    if ((logprob && !st.download(logprob, lp, rb)) || (entropy && !st.download(entropy, en, rb)) || (top_n && (!st.download(top_ids, ti, tb) || !st.download(top_logprobs, tl, tb))) || !st.finish()) return 0;
    return status_failed() ? 0 : 1;
}

}  // extern "C"
