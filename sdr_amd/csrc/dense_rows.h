// Sparse rows of ids against dense matrices: what the kernels of lookup.hip, lookup_grad.hip and winners.hip share.
#pragma once

#include <type_traits>

#include "sdrb_internal.h"

namespace sdrb {

// ---- element types: SDRB_F32 / SDRB_F16 / SDRB_BF16, arithmetic always in binary32 or wider ----
using f16 = _Float16;
using bf16 = __bf16;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(f16 v) { return (float)v; }
__device__ __forceinline__ float to_f32(bf16 v) { return (float)v; }
// round to nearest even, the one rounding of a result to its type
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
    return (T)v;
}

// 16, 8 and 4 bytes at any multiple of two: the unaligned access mode of the target makes each one load or store
using Bytes16 = uint32_t __attribute__((ext_vector_type(4), aligned(2)));
using Bytes8 = uint32_t __attribute__((ext_vector_type(2), aligned(2)));
using Bytes4 = uint32_t __attribute__((ext_vector_type(1), aligned(2)));
template <int BYTES>
using Bytes = std::conditional_t<BYTES % 16 == 0, Bytes16, std::conditional_t<BYTES % 8 == 0, Bytes8, Bytes4>>;

// N consecutive elements starting at any multiple of the element's own size
template <int N, typename T>
__device__ __forceinline__ void load_n(const T* p, T (&t)[N]) {
    if constexpr (N * sizeof(T) % 4 == 0) {
        using B = Bytes<(int)(N * sizeof(T))>;
#pragma unroll
        for (size_t k = 0; k < N * sizeof(T) / sizeof(B); ++k) {
            const B raw = reinterpret_cast<const B*>(p)[k];
            __builtin_memcpy(reinterpret_cast<char*>(t) + k * sizeof(B), &raw, sizeof(B));
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) t[k] = p[k];
    }
}
template <int N, typename T, std::enable_if_t<!std::is_same_v<T, float>, int> = 0>
__device__ __forceinline__ void load_n(const T* p, float (&v)[N]) {
    T t[N];
    load_n<N>(p, t);
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = to_f32(t[k]);
}
template <int N, typename T>
__device__ __forceinline__ void store_n(T* p, const float (&v)[N]) {
    T t[N];
#pragma unroll
    for (int k = 0; k < N; ++k) t[k] = from_f32<T>(v[k]);
    if constexpr (N * sizeof(T) % 4 == 0) {
        using B = Bytes<(int)(N * sizeof(T))>;
#pragma unroll
        for (size_t k = 0; k < N * sizeof(T) / sizeof(B); ++k) {
            B raw;
            __builtin_memcpy(&raw, reinterpret_cast<const char*>(t) + k * sizeof(B), sizeof(B));
            reinterpret_cast<B*>(p)[k] = raw;
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) p[k] = t[k];
    }
}

// ---- values moved between the lanes of a wave, without LDS ----
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp(uint32_t other, uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)other, (int)v, CTRL, ROWS, 0xF, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp(float other, float v) {
    return __builtin_bit_cast(float, dpp<CTRL, ROWS>(__builtin_bit_cast(uint32_t, other), __builtin_bit_cast(uint32_t, v)));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp(double other, double v) {
    const uint64_t o = __builtin_bit_cast(uint64_t, other), x = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = dpp<CTRL, ROWS>((uint32_t)o, (uint32_t)x), hi = dpp<CTRL, ROWS>((uint32_t)(o >> 32), (uint32_t)(x >> 32));
    return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
// inclusive sums over the lanes of a wave, or of each row of 16
template <int LANES>
__device__ __forceinline__ uint32_t scan_lanes(uint32_t v) {
    v += dpp<0x111, 0xF>(0u, v);   // one lane up in a row of 16, two, four, eight
    v += dpp<0x112, 0xF>(0u, v);
    v += dpp<0x114, 0xF>(0u, v);
    v += dpp<0x118, 0xF>(0u, v);
    if constexpr (LANES == 64) {
        v += dpp<0x142, 0xA>(0u, v);   // lane 15 of the row of 16 below, into rows 1 and 3
        v += dpp<0x143, 0xC>(0u, v);   // lane 31, into rows 2 and 3
    }
    return v;
}

// The segment that holds element p is the last one whose first element is at or before p.  A wave looks at 64
// segments a step.
__device__ __forceinline__ uint64_t segment_at(const uint32_t* __restrict__ start, uint64_t n_segments, uint64_t p) {
    uint64_t lo = 0, n = n_segments;   // it is one of [lo, lo + n)
    while (n > 1) {
        const uint64_t stride = (n + 63) / 64, at = lo + (threadIdx.x & 63) * stride;
        const bool reached = at < lo + n && start[at] <= p;
        const uint64_t last = (uint64_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64(reached));   // lane 0 always, unless p is before all
        const uint64_t step = last ? (last - 1) * stride : 0;
        n = n - step < stride ? n - step : stride;
        lo += step;
    }
    return lo;
}

// Calls f(T{}) with the element type named by `type` (checked by the caller).
template <typename F>
int with_type(int type, F&& f) {
    switch (type) {
        case SDRB_F16: return f(f16{});
        case SDRB_BF16: return f(bf16{});
        default: return f(float{});
    }
}
// more than 64 KiB of LDS, all in all, has to be asked for
template <typename F>
int allow_lds(F* kernel, size_t dynamic_bytes) {
    if (dynamic_bytes > 49152)
        SDRB_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)dynamic_bytes));
    return SDRB_OK;
}
// A launch takes fewer than 2^32 threads: more blocks become several launches.  go(first block, blocks)
template <typename F>
int in_launches(uint64_t blocks, uint32_t threads, F&& go) {
    const uint64_t most = 0xFFFFFFFFu / threads / 64 * 64;
    for (uint64_t first = 0; first < blocks; first += most) {
        const int rc = go(first, (uint32_t)(blocks - first < most ? blocks - first : most));
        if (rc != SDRB_OK) return rc;
    }
    return SDRB_OK;
}
inline size_t type_size(int type) { return type == SDRB_F32 ? 4 : 2; }

// A ragged sum: out[s, :] (+)= scale * sum over the elements p of segment s of weight[p] * src[index[p], :].
// lookup.hip runs it over a batch's rows, lookup_grad.hip over the elements sorted by id.
struct GatherSum {
    uint64_t n_segments;
    uint64_t n_elems;
    const uint32_t* start;     // [n_segments + 1], or null: every segment holds n_elems / n_segments elements
    // or, with keys given: segments are the runs of equal keys of a sorted list, n_segments is n_elems, and a run's sum goes to
    // the row of out that its key names (a key of out_rows or more: none); a run's first element and the one after its last
    const uint32_t *keys, *begin, *end;
    uint64_t out_rows;
    const void* index;         // [n_elems]
    int index_bits;            // 32 or 64; an index outside [0, src_rows) contributes nothing
    const float* weight;       // [n_elems] or null: 1
    const void* src;
    int src_type;
    uint64_t src_rows, src_ld;
    uint32_t dim;
    void* out;
    int out_type;
    uint64_t out_ld;
    float scale;
    bool accumulate;           // segments without elements are then left as they are
    uint32_t chunk;            // segments longer than this are summed in two steps (0: all in one) ...
    float* partials;           // ... the first of which leaves its sums here: partial_bytes(...)
};
// A chunk for ragged segments or equal ones; 0: none is longer, or each is summed by a whole block.
uint32_t segment_chunk(uint64_t n_segments, uint64_t n_elems, uint32_t dim, bool ragged);
uint32_t run_chunk(uint64_t n_elems);
inline size_t partial_bytes(uint32_t chunk, uint64_t n_elems, uint32_t dim) {
    return chunk ? (size_t)((n_elems + chunk - 1) / chunk) * 2 * dim * sizeof(float) : 0;
}
int launch_gather_sum(const GatherSum& g, hipStream_t stream);

// lookup_grad.hip
size_t table_grad_scratch_bytes(const sdrb_rows& rows, uint64_t n_table_rows, uint32_t dim);
int launch_table_grad(const sdrb_rows& rows, const sdrb_dense& grad, float scale, bool accumulate,
                      const sdrb_dense& out, void* scratch, hipStream_t stream);
int launch_weight_grad(const sdrb_rows& rows, const sdrb_dense& grad, const sdrb_dense& table, float scale, float* out,
                       hipStream_t stream);

// winners.hip
constexpr uint32_t kWinnersMaxIds = 16384, kWinnersMaxK = 1024, kWinnersMaxGroups = 256;
int launch_winners(const sdrb_dense& scores, const sdrb_winners_spec& spec, int32_t* ids, float* weights, hipStream_t stream);
int launch_winners_grad(const sdrb_dense& scores, const sdrb_winners_spec& spec, const int32_t* ids, const float* grad_weights,
                        const sdrb_dense& out, hipStream_t stream);

}  // namespace sdrb
