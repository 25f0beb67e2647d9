// The value types of the batch operators' rows (F32, F16, BF16 by ggml id): loads as floats, stores rounded to nearest even, and what their
// entry points check on the host.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "redcuda_common.cuh"

namespace rc {

constexpr uint32_t VT_F32 = 0u, VT_F16 = 1u, VT_BF16 = 30u;       // ggml ids
inline uint32_t val_size(uint32_t t) { return t == VT_F32 ? 4u : t == VT_F16 || t == VT_BF16 ? 2u : 0u; }

inline bool aligned16(const void *p) { return ((uintptr_t)p & 15u) == 0; }
inline bool aligned4(const void *p) { return ((uintptr_t)p & 3u) == 0; }
inline bool overlap(const void *a, uint64_t na, const void *b, uint64_t nb) {
    return a && b && na && nb && (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na;
}
struct Span { const void *p; uint64_t n; };
// whether an array that is written lies in one that is read or in another that is written
template <int W, int R> inline bool spans_overlap(const Span (&written)[W], const Span (&read)[R]) {
    for (int i = 0; i < W; ++i) {
        for (int j = 0; j < R; ++j) if (overlap(written[i].p, written[i].n, read[j].p, read[j].n)) return true;
        for (int j = 0; j < i; ++j) if (overlap(written[i].p, written[i].n, written[j].p, written[j].n)) return true;
    }
    return false;
}
// bytes of `rows` rows of n elements that lie `stride` elements apart
inline uint64_t span_bytes(uint64_t rows, uint64_t stride, uint64_t n, uint32_t size) { return rows ? ((rows - 1u) * stride + n) * size : 0u; }
// streaming multiprocessors of the current device (0: unknown)
inline uint32_t sm_count() {
    static std::atomic<uint32_t> known[64];
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0u;
    uint32_t c = known[dev].load(std::memory_order_relaxed);
    if (!c && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess) known[dev].store(c = (uint32_t)n, std::memory_order_relaxed);
    return c;
}

// raises a kernel's limit of dynamic shared memory once per device; set: a bit for each device on which that has been done
inline int raise_smem_limit(const void *kernel, size_t bytes, std::atomic<uint64_t> &set) {
    int dev = 0;
    RC_CUDA(cudaGetDevice(&dev));
    if (dev < 64 && (set.load(std::memory_order_relaxed) >> dev & 1u)) return 1;
    RC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    if (dev < 64) set.fetch_or(1ull << dev, std::memory_order_relaxed);
    return 1;
}

#ifdef __CUDACC__
__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// N neighbouring values, aligned to N values
template <class T, int N> struct alignas(sizeof(T) * N) Pack { T v[N]; };
template <int N, class T> __device__ __forceinline__ void load_vals(const T *p, float (&x)[N]) {
    static_assert(N * sizeof(T) <= 16, "one load");
    const Pack<T, N> a = *reinterpret_cast<const Pack<T, N> *>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = to_f32(a.v[i]);
}
template <int N, class T> __device__ __forceinline__ void store_vals(T *p, const float (&x)[N]) {
    static_assert(N * sizeof(T) <= 16, "one store");
    Pack<T, N> a;
#pragma unroll
    for (int i = 0; i < N; ++i) a.v[i] = from_f32<T>(x[i]);
    *reinterpret_cast<Pack<T, N> *>(p) = a;
}

// whether the bounds of sequence b ascend within n rows
__device__ __forceinline__ bool seq_bounds(const int32_t *cu, uint32_t b, uint32_t n) {
    const int32_t lo = cu[b], hi = cu[b + 1u];
    return lo >= 0 && hi >= lo && (uint32_t)hi <= n;
}
// The sequence with right bounds that row t of n belongs to, found by a whole warp; n_seqs: none. Ascending bounds are searched 32 at a step. Where that gives no such sequence (the row is of none,
// or some bound is wrong and the search was led astray) all are looked at, 32 at a time: 256 sequences are eight reads that do not wait for one another.
__device__ __forceinline__ uint32_t find_seq(const int32_t *cu, uint32_t n_seqs, uint32_t t, uint32_t n) {
    const uint32_t lane = threadIdx.x & 31u;
    uint32_t lo = 0u, cnt = n_seqs;              // entries lo .. lo + cnt - 1 are open
    while (cnt > 1u) {
        const uint32_t step = (cnt + 31u) / 32u, i = lane * step, m = __ballot_sync(0xffffffffu, i < cnt && cu[lo + i] <= (int32_t)t), at = (m ? 31u - (uint32_t)__clz((int)m) : 0u) * step;
        cnt = min(step, cnt - at); lo += at;
    }
    auto has = [&](uint32_t b) { return seq_bounds(cu, b, n) && (int32_t)t >= cu[b] && (int32_t)t < cu[b + 1u]; };
    if (has(lo)) return lo;
    for (uint32_t b = 0u; b < n_seqs; b += 32u) {
        const uint32_t m = __ballot_sync(0xffffffffu, b + lane < n_seqs && has(b + lane));
        if (m) return b + (uint32_t)__ffs((int)m) - 1u;
    }
    return n_seqs;
}
#endif

}  // namespace rc
