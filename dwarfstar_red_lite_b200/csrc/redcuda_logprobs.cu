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
#include <type_traits>

namespace rc {

namespace cg = cooperative_groups;

constexpr int LP_WARPS = 8, LP_CLUSTER = 8, LP_UNROLL = 4;
static_assert(REDCUDA_MAX_ALTERNATIVES <= 32u && LP_WARPS == 8 && LP_CLUSTER == LP_WARPS, "a list is one key a lane; eight floors are read at once; a warp for every list");

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

__device__ __forceinline__ float max_nan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float exp2_fast(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }      // 2 units

__device__ __forceinline__ float4 lp_floor(const float *s) {                 // other warps write it meanwhile
    float4 r;
    asm volatile("ld.volatile.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(r.x), "=f"(r.y), "=f"(r.z), "=f"(r.w) : "r"((uint32_t)__cvta_generic_to_shared(s)));
    return r;
}

// 32 keys, one a lane, in two networks: any order to descending, and the 32 largest of two descending lists.
__device__ __forceinline__ uint64_t lp_exchange(uint64_t key, int w, bool larger) {
    const uint64_t other = __shfl_xor_sync(0xffffffffu, key, w);
    return (key > other) == larger ? key : other;
}
__device__ __forceinline__ uint64_t lp_sort(uint64_t key) {
    const uint32_t lane = threadIdx.x & 31u;
#pragma unroll
    for (uint32_t run = 2; run <= 32; run <<= 1)
#pragma unroll
        for (uint32_t w = run >> 1; w; w >>= 1) key = lp_exchange(key, (int)w, ((lane & w) == 0u) == ((lane & run) == 0u || run == 32u));
    return key;
}
__device__ __forceinline__ uint64_t lp_merge(uint64_t a, uint64_t b) {       // both descending
    const uint32_t lane = threadIdx.x & 31u;
    const uint64_t r = __shfl_sync(0xffffffffu, b, 31 - (int)lane);
    uint64_t key = a > r ? a : r;
#pragma unroll
    for (uint32_t w = 16; w; w >>= 1) key = lp_exchange(key, (int)w, (lane & w) == 0u);
    return key;
}

// Sixteen bytes of logits as floats, and the largest of them (a NaN counts as none)
__device__ __forceinline__ void lp_unpack(uint4 w, float (&v)[4]) { v[0] = __uint_as_float(w.x); v[1] = __uint_as_float(w.y); v[2] = __uint_as_float(w.z); v[3] = __uint_as_float(w.w); }
template <class T> __device__ __forceinline__ void lp_unpack(uint4 w, float (&v)[8]) {
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<T, __half>::value) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&x[i]));
            v[2 * i] = f.x; v[2 * i + 1] = f.y;
        } else {
            v[2 * i] = __uint_as_float(x[i] << 16); v[2 * i + 1] = __uint_as_float(x[i] & 0xffff0000u);
        }
    }
}
template <class T> __device__ __forceinline__ float lp_most(uint4 w) {
    if constexpr (sizeof(T) == 4) {
        return fmaxf(fmaxf(fmaxf(__uint_as_float(w.x), __uint_as_float(w.y)), fmaxf(__uint_as_float(w.z), __uint_as_float(w.w))), -INFINITY);
    } else {
        using P = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
        auto pair = [](const uint32_t &x) { return *reinterpret_cast<const P *>(&x); };
        const P m = __hmax2(__hmax2(pair(w.x), pair(w.y)), __hmax2(pair(w.z), pair(w.w)));
        return fmaxf(fmaxf(to_f32(m.x), to_f32(m.y)), -INFINITY);
    }
}

// What bounds it is the row's bytes for 32-bit logits (592 rows of 151936: 56 us, 6.4 TB/s) and instructions for 16-bit ones (seven a value, one of them an exponential at a
// sixteenth of the fp32 rate: 777 rows 50 us, 4.8 TB/s). A round's loads are on their way while the last one's values are added up; four blocks an SM for 32 bits, three for 16, which have to
// spill more with four (777 rows 65 us); as they are, each of the three forms spills one register.
// The alternatives cost one comparison a lane and round of LP_UNROLL pieces where there are none: a warp keeps its 32 largest keys, one a
// lane, and looks at single values only where the largest of a lane's round reaches what is known to be among the row's n largest. That is the n-th of the warp's own,
// or the least of the warps' ceil(n / LP_WARPS)-th largest, which every warp publishes (n values are at least that large; a stale one is a lower bound too), or in a warp's first
// round the n-th of its lanes' largest. 777 rows of BF16 with 5, 20 alternatives: 69, 82 us (the n-th of what the warps publish instead of the least, found anew with every list: 69, 93).
template <class T>
__global__ void __launch_bounds__(LP_WARPS * 32, sizeof(T) == 4 ? 4 : 3) k_token_logprobs(LogprobArgs A) {
    pdl_prologue();
    constexpr int VEC = 16 / sizeof(T), U = LP_UNROLL;
    constexpr float LOG2E = 1.44269504088896340736f;
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t parts = cluster.num_blocks(), part = cluster.block_rank(), row = blockIdx.x / parts;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, n = A.top_n;
    __shared__ uint64_t s_keys[LP_WARPS][32], s_best[LP_CLUSTER][32];
    __shared__ LpSums s_sums[LP_WARPS], s_parts[LP_CLUSTER];
    __shared__ __align__(16) float s_floor[LP_WARPS];
    const T *x = reinterpret_cast<const T *>(A.x) + (uint64_t)row * A.row_stride;
    // the row as up to VEC - 1 single values, whole 16-byte pieces, up to VEC - 1 single values
    const uint32_t head = min(A.vocab, (uint32_t)((16u - ((uintptr_t)x & 15u)) & 15u) / (uint32_t)sizeof(T)), pieces = (A.vocab - head) / VEC;
    const uint32_t per = (pieces + parts - 1u) / parts, p0 = min(pieces, part * per), p1 = min(pieces, p0 + per);
    if (lane == 0u) s_floor[warp] = -INFINITY;
    __syncthreads();

    float m = -INFINITY;                         // a lane's sums are kept in two halves each
    float2 s2 = make_float2(0.f, 0.f), u2 = make_float2(0.f, 0.f);
    uint64_t best = 0ull, least = 0ull;          // lane i: the i-th largest key; the n-th
    float bar = -INFINITY;                       // values below it are not among the row's n largest
    const uint32_t share = (n + LP_WARPS - 1u) / LP_WARPS;
    auto listed = [&]() {                        // the list has changed
        least = __shfl_sync(0xffffffffu, best, (int)n - 1);
        const uint64_t mine = __shfl_sync(0xffffffffu, best, (int)share - 1);
        if (lane == 0u) reinterpret_cast<volatile float *>(s_floor)[warp] = mine ? lp_value(mine) : -INFINITY;
    };
    auto offer = [&](uint64_t key) {             // a key of each lane, 0: none
        uint32_t todo = __ballot_sync(0xffffffffu, key > least);
        if (!todo) return;
        if (__popc(todo) > 6) {
            best = lp_merge(best, lp_sort(key));
        } else {
            for (; todo; todo &= todo - 1u) {
                const uint64_t k = __shfl_sync(0xffffffffu, key, (int)__ffs((int)todo) - 1), up = __shfl_up_sync(0xffffffffu, best, 1);
                best = best >= k ? best : lane == 0u || up >= k ? k : up;
            }
        }
        listed();
    };
    auto rescale = [&](float to) {
        const float f = to > m ? exp2_fast(max_nan(m - to, -150.f) * LOG2E) : 1.f, d = m == -INFINITY ? 0.f : m - to;
        u2 = make_float2(f > 0.f ? f * (u2.x + s2.x * d) : 0.f, f > 0.f ? f * (u2.y + s2.y * d) : 0.f);
        s2.x *= f; s2.y *= f;
        m = to;
    };
    // the token and its logit are asked for long before they are wanted: read at the end, one after the other, they would take a microsecond of every row
    const bool asks = A.logprob && part == 0u && tid == 0u;
    int32_t token = -1;
    if (asks) asm volatile("ld.global.nc.s32 %0, [%1];" : "=r"(token) : "l"(A.tokens + row));
    bool fresh = true;
    uint4 ahead[U];                              // the next round's pieces
    auto load = [&](uint32_t p) {
        const uint4 *const at = reinterpret_cast<const uint4 *>(x + head) + p + lane;
        if (p + 32u * U <= p1) {
#pragma unroll
            for (int u = 0; u < U; ++u) ahead[u] = at[u * 32];
        } else {
            const uint32_t low = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;       // -infinity
#pragma unroll
            for (int u = 0; u < U; ++u) ahead[u] = p + u * 32u + lane < p1 ? at[u * 32] : make_uint4(low, low, low, low);
        }
    };
    load(p0 + warp * (32u * U));
    for (uint32_t p = p0 + warp * (32u * U); p < p1; p += LP_WARPS * 32u * U) {
        uint4 w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) w[u] = ahead[u];
        load(p + LP_WARPS * 32u * U);
        float top[U], most = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; ++u) { top[u] = lp_most<T>(w[u]); most = fmaxf(most, top[u]); }
        if (__any_sync(0xffffffffu, most > m)) rescale(fmaxf(m, most));
        const float base = m == -INFINITY ? 0.f : m;
        const float2 nb = make_float2(-base, -base), l2 = make_float2(LOG2E, LOG2E);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float v[VEC];
            if constexpr (sizeof(T) == 4) lp_unpack(w[u], v); else lp_unpack<T>(w[u], v);
#pragma unroll
            for (int i = 0; i < VEC; i += 2) {
                float2 d = __fadd2_rn(make_float2(v[i], v[i + 1]), nb);
                d = make_float2(max_nan(d.x, -150.f), max_nan(d.y, -150.f));       // of a probability that is 0, e d = 0; of a NaN, a NaN
                float2 e = __fmul2_rn(d, l2);
                e = make_float2(exp2_fast(e.x), exp2_fast(e.y));
                s2 = __fadd2_rn(s2, e);
                u2 = __ffma2_rn(e, d, u2);
            }
        }
        if (n == 0u) continue;
        const float4 f0 = lp_floor(&s_floor[0]), f1 = lp_floor(&s_floor[4]);
        // Other warps write the floors meanwhile, and a 16-byte read of a warp is not one access: its lanes may see different ones. One lane's is taken, as the warp branches on it.
        bar = __shfl_sync(0xffffffffu, fmaxf(bar, fminf(fminf(fminf(f0.x, f0.y), fminf(f0.z, f0.w)), fminf(fminf(f1.x, f1.y), fminf(f1.z, f1.w)))), 0);
        if (fresh) {                             // the n-th of the lanes' largest
            fresh = false;
            float y = most;
#pragma unroll
            for (uint32_t run = 2; run <= 32; run <<= 1)
#pragma unroll
                for (uint32_t k = run >> 1; k; k >>= 1) {
                    const float o = __shfl_xor_sync(0xffffffffu, y, k);
                    y = ((lane & k) == 0u) == ((lane & run) == 0u || run == 32u) ? fmaxf(y, o) : fminf(y, o);
                }
            bar = fmaxf(bar, __shfl_sync(0xffffffffu, y, (int)n - 1));
        }
        // what equals the n-th of earlier rounds has a larger index
        if (!__any_sync(0xffffffffu, most >= bar && (least == 0ull || most > lp_value(least)))) continue;
        // a lane's values that reach the bar, as bits, which are then offered one a lane at a time
        static_assert(U * VEC <= 32, "a bit each");
        uint32_t places = 0u;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (!__any_sync(0xffffffffu, top[u] >= bar)) continue;
            float v[VEC];
            if constexpr (sizeof(T) == 4) lp_unpack(w[u], v); else lp_unpack<T>(w[u], v);
            if (p + u * 32u + lane < p1)
#pragma unroll
                for (int i = 0; i < VEC; ++i) places |= v[i] >= bar ? 1u << (u * VEC + i) : 0u;
        }
#pragma unroll 1
        while (__any_sync(0xffffffffu, places)) {
            uint64_t key = 0ull;
            if (places) {
                const uint32_t j = (uint32_t)__ffs((int)places) - 1u, i = head + (p + j / VEC * 32u + lane) * VEC + j % VEC;
                places &= places - 1u;
                key = lp_key(to_f32(x[i]), i);
            }
            offer(key);
        }
        if (least) bar = fmaxf(bar, lp_value(least));
    }
    if (part == 0u && warp == 0u) {              // the single values at both ends
        const uint32_t tail = head + pieces * VEC, ends = head + A.vocab - tail;
        const uint32_t i = lane < head ? lane : tail + lane - head;
        const bool have = lane < ends;
        const float v = have ? to_f32(x[i]) : -INFINITY;
        if (v > m) rescale(v);
        const float d = max_nan(v - (m == -INFINITY ? 0.f : m), -150.f), e = exp2_fast(d * LOG2E);
        s2.x += e;
        u2.x += e * d;
        if (n) offer(have && v == v ? lp_key(v, i) : 0ull);
    }
    const bool known = token >= 0 && (uint32_t)token < A.vocab;
    T logit = from_f32<T>(0.f);
    if (asks && known) logit = x[token];
    LpSums S{m, s2.x + s2.y, u2.x + u2.y};
#pragma unroll
    for (int w = 16; w; w >>= 1) {
        const LpSums o{__shfl_xor_sync(0xffffffffu, S.m, w), __shfl_xor_sync(0xffffffffu, S.s, w), __shfl_xor_sync(0xffffffffu, S.u, w)};
        S = lp_join(S, o);
    }
    if (lane == 0u) s_sums[warp] = S;
    s_keys[warp][lane] = best;
    // the lists of a block, and then of a cluster, two and two
    auto gather = [&](uint64_t (&list)[LP_WARPS][32], uint32_t lists) {
        for (uint32_t half = LP_WARPS / 2; half; half >>= 1) {
            if (warp < half && warp + half < lists) { best = lp_merge(best, list[warp + half][lane]); list[warp][lane] = best; }
            __syncthreads();
        }
    };
    __syncthreads();
    if (n) gather(s_keys, LP_WARPS);
    if (parts > 1u) cluster.sync();              // the other blocks have begun: their shared memory may be written
    if (warp == 0u) {
        S = lane < LP_WARPS ? s_sums[lane] : LpSums{-INFINITY, 0.f, 0.f};
#pragma unroll
        for (int w = LP_WARPS / 2; w; w >>= 1) {
            const LpSums o{__shfl_xor_sync(0xffffffffu, S.m, w), __shfl_xor_sync(0xffffffffu, S.s, w), __shfl_xor_sync(0xffffffffu, S.u, w)};
            S = lp_join(S, o);
        }
        if (parts > 1u) {
            if (n) cluster.map_shared_rank(s_best[part], 0)[lane] = best;
            if (lane == 0u) *cluster.map_shared_rank(&s_parts[part], 0) = S;
        }
    }
    if (parts > 1u) {
        cluster.sync();
        if (part != 0u) return;
        if (n) {
            best = warp < parts ? s_best[warp][lane] : 0ull;
            gather(s_best, parts);
        }
    }
    if (warp != 0u) return;
    if (parts > 1u) {
        S = lane < parts ? s_parts[lane] : LpSums{-INFINITY, 0.f, 0.f};
#pragma unroll
        for (int w = LP_CLUSTER / 2; w; w >>= 1) {
            const LpSums o{__shfl_xor_sync(0xffffffffu, S.m, w), __shfl_xor_sync(0xffffffffu, S.s, w), __shfl_xor_sync(0xffffffffu, S.u, w)};
            S = lp_join(S, o);
        }
    }
    S.m = __shfl_sync(0xffffffffu, S.m, 0); S.s = __shfl_sync(0xffffffffu, S.s, 0); S.u = __shfl_sync(0xffffffffu, S.u, 0);
    const float ls = logf(S.s);                  // nothing left: m = -infinity, s = 0
    const bool nan = !(S.s == S.s), none = !nan && S.m == -INFINITY;
    if (lane == 0u) {
        if (A.logprob) {
            float lp = NAN;
            if (known) lp = nan ? NAN : none ? -INFINITY : (to_f32(logit) - S.m) - ls;
            else if (token != -1 && A.status) A.status[ST_TOKEN_RANGE] = 1u;
            A.logprob[row] = lp;
        }
        if (A.entropy) A.entropy[row] = nan ? NAN : none ? 0.f : fmaxf(ls - S.u / S.s, 0.f);
    }
    if (lane < n) {
        A.top_ids[(uint64_t)row * n + lane] = nan ? -1 : (int32_t)~(uint32_t)best;
        A.top_lp[(uint64_t)row * n + lane] = nan ? NAN : none ? -INFINITY : (lp_value(best) - S.m) - ls;
    }
}

template <class T> static int launch_logprobs(const LogprobArgs &A, uint32_t rows, cudaStream_t s) {
    const uint32_t sms = sm_count();
    uint32_t parts = 1u;
    // Blocks of a row: until there are two for every SM. Twice as many change nothing for up to 36 rows (24 us for 36 of 152064 F16 logits), 145 rows of F32 take 35 -> 41 us; eight times
    // as many 777 rows of BF16 101 -> 140: a block's end costs some 4 us.
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
    const Span written[4] = {{logprob_dev, ob}, {entropy_dev, ob}, {top_ids_dev, ob * top_n}, {top_logprobs_dev, ob * top_n}}, read[2] = {{logits_dev, lb}, {tokens_dev, ob}};
    RC_REQUIRE(!spans_overlap(written, read), "token logprobs: an output lies inside the logits, the tokens or another output");
    RC_REQUIRE(aligned4(tokens_dev) && aligned4(logprob_dev) && aligned4(entropy_dev) && aligned4(top_ids_dev) && aligned4(top_logprobs_dev), "token logprobs: tokens or outputs are not 4-byte aligned");
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
