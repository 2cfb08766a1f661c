// Ragged gather-sums over a dense matrix: out[s, :] = scale * sum of weight[p] * src[index[p], :] over a segment's
// elements p.  A lookup runs it over the rows of a batch, the table's gradient over the elements sorted by id.
//
// A group of lanes owns one segment and one slice of the columns, 16 bytes of src a lane, and adds the segment's
// elements in order into binary32 registers; the sum is scaled and rounded once to the output's type.  A segment of
// more than `chunk` elements would keep its group busy long after the others: its elements are summed by groups that
// own a chunk of the element list each (k_gather_chunks), and the segment's own group adds those sums up in order.
// Every order of additions follows from the shapes and offsets alone: results repeat bit for bit.
#include <algorithm>

#include "dense_rows.h"

namespace sdrb {

namespace {

struct GatherArgs {
    uint64_t n_segments, n_elems, src_rows, src_ld, out_ld;
    const uint32_t* start;
    const float* weight;
    float* partials;
    float scale;
    uint32_t row_len;       // where start is null
    uint32_t dim;
    uint32_t chunk;         // longer segments come from `partials` (0: there are none)
    uint32_t lanes_log2;    // lanes of a group
    uint32_t slices;        // of the columns
};

// the elements [lo, hi) of a segment; offsets that run backwards or past the list are cut to it
__device__ __forceinline__ void segment_of(const GatherArgs& a, uint64_t s, uint64_t& lo, uint64_t& hi) {
    if (a.start) {
        lo = a.start[s];
        hi = a.start[s + 1];
        hi = hi < a.n_elems ? hi : a.n_elems;
        lo = lo < hi ? lo : hi;
    } else {
        lo = s * a.row_len;
        hi = lo + a.row_len;
    }
}

template <int V, typename T, typename Id, bool WEIGHTED>
__device__ __forceinline__ void add_elements(const GatherArgs& a, const Id* __restrict__ index, const T* __restrict__ src,
                                             uint64_t lo, uint64_t hi, uint32_t col, float (&acc)[V]) {
    for (uint64_t p = lo; p < hi; ++p) {
        const Id id = index[p];
        if (id < 0 || (uint64_t)id >= a.src_rows) continue;
        float v[V];
        load_n<V>(src + (uint64_t)id * a.src_ld + col, v);
        const float w = WEIGHTED ? a.weight[p] : 1.0f;
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] = WEIGHTED ? fmaf(w, v[k], acc[k]) : acc[k] + v[k];
    }
}

// Where a group stands: its segment (or chunk) and the first column of this lane.  A lane whose columns would run past
// the end reads the last V columns instead and stores only what is its own (from `col_own`).
struct Place {
    uint64_t item;
    uint32_t slice, col, col_own;
    bool live;
};
template <int V>
__device__ __forceinline__ Place place_of(const GatherArgs& a, uint64_t n_items) {
    Place p;
    const uint32_t groups = 256u >> a.lanes_log2, group = threadIdx.x >> a.lanes_log2;
    const uint32_t lane = threadIdx.x & ((1u << a.lanes_log2) - 1u);
    p.slice = blockIdx.x % a.slices;
    p.item = (uint64_t)(blockIdx.x / a.slices) * groups + group;
    p.col_own = ((p.slice << a.lanes_log2) + lane) * V;
    p.live = p.item < n_items && p.col_own < a.dim;
    p.col = p.col_own + V <= a.dim ? p.col_own : a.dim - V;
    return p;
}

template <int V, typename T, typename O, typename Id, bool WEIGHTED, bool ACCUMULATE>
__global__ __launch_bounds__(256) void k_gather_rows(GatherArgs a, const Id* __restrict__ index, const T* __restrict__ src,
                                                     O* __restrict__ out) {
    const Place at = place_of<V>(a, a.n_segments);
    if (!at.live) return;
    uint64_t lo, hi;
    segment_of(a, at.item, lo, hi);
    if (ACCUMULATE && lo == hi) return;
    float acc[V];
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] = 0.0f;
    if (a.chunk && hi - lo > a.chunk) {
        // chunk c of the element list keeps two sums: of the segment its first element lies in, and of the one its last
        for (uint64_t c = lo / a.chunk; c * a.chunk < hi; ++c) {
            const float* part = a.partials + (2 * c + (c * a.chunk < lo ? 1 : 0)) * a.dim + at.col;
            float v[V];
            load_n<V>(part, v);
#pragma unroll
            for (int k = 0; k < V; ++k) acc[k] += v[k];
        }
    } else {
        add_elements<V, T, Id, WEIGHTED>(a, index, src, lo, hi, at.col, acc);
    }
    O* to = out + at.item * a.out_ld + at.col;
    if (at.col == at.col_own) {
        if (ACCUMULATE) {
            float old[V];
            load_n<V>(to, old);
#pragma unroll
            for (int k = 0; k < V; ++k) acc[k] = fmaf(a.scale, acc[k], old[k]);
        } else {
#pragma unroll
            for (int k = 0; k < V; ++k) acc[k] *= a.scale;
        }
        store_n<V>(to, acc);
    } else {
        const uint32_t skip = at.col_own - at.col;
#pragma unroll
        for (int k = 0; k < V; ++k)
            if ((uint32_t)k >= skip) to[k] = from_f32<O>(ACCUMULATE ? fmaf(a.scale, acc[k], to_f32(to[k])) : acc[k] * a.scale);
    }
}

// last segment whose first element is at or before p (p < n_elems): the one that holds p, empty segments being passed over
__device__ __forceinline__ uint64_t segment_at(const uint32_t* __restrict__ start, uint64_t n_segments, uint64_t p) {
    uint64_t lo = 0, hi = n_segments;
    while (hi - lo > 1) {
        const uint64_t mid = (lo + hi) >> 1;
        if (start[mid] <= p) lo = mid;
        else hi = mid;
    }
    return lo;
}

// the sums that chunk c of the element list contributes to segments longer than a chunk
template <int V, typename T, typename Id, bool WEIGHTED>
__global__ __launch_bounds__(256) void k_gather_chunks(GatherArgs a, const Id* __restrict__ index, const T* __restrict__ src,
                                                       uint64_t n_chunks) {
    const Place at = place_of<V>(a, n_chunks);
    if (!at.live) return;
    const uint64_t c_lo = at.item * a.chunk, c_hi = c_lo + a.chunk < a.n_elems ? c_lo + a.chunk : a.n_elems;
#pragma unroll
    for (int end = 0; end < 2; ++end) {
        uint64_t lo, hi;
        if (a.start) {
            segment_of(a, segment_at(a.start, a.n_segments, end ? c_hi - 1 : c_lo), lo, hi);
        } else {
            lo = (end ? c_hi - 1 : c_lo) / a.row_len * a.row_len;
            hi = lo + a.row_len;
        }
        if (hi - lo <= a.chunk) continue;
        if (end && lo <= c_lo) continue;   // the first element's segment once more
        float acc[V];
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] = 0.0f;
        add_elements<V, T, Id, WEIGHTED>(a, index, src, lo > c_lo ? lo : c_lo, hi < c_hi ? hi : c_hi, at.col, acc);
        float* to = a.partials + (2 * at.item + end) * a.dim + at.col;
        if (at.col == at.col_own) {
            store_n<V>(to, acc);
        } else {
            const uint32_t skip = at.col_own - at.col;
#pragma unroll
            for (int k = 0; k < V; ++k)
                if ((uint32_t)k >= skip) to[k] = acc[k];
        }
    }
}

// the longest run of elements that one group of lanes sums by itself
uint32_t chunk_of(uint64_t n_segments, uint64_t n_elems) {
    const uint64_t mean = n_elems / (n_segments ? n_segments : 1);
    uint32_t chunk = 128;
    while (chunk < 4 * mean && chunk < 1024) chunk *= 2;
    return chunk;
}

template <int V, typename T, typename O, typename Id, bool WEIGHTED>
int launch_typed(const GatherSum& g, GatherArgs a, hipStream_t stream) {
    const Id* index = static_cast<const Id*>(g.index);
    const T* src = static_cast<const T*>(g.src);
    uint32_t lanes_log2 = 0;
    while (lanes_log2 < 6 && ((uint64_t)V << lanes_log2) < a.dim) ++lanes_log2;
    a.lanes_log2 = lanes_log2;
    a.slices = (uint32_t)((a.dim + ((uint64_t)V << lanes_log2) - 1) / ((uint64_t)V << lanes_log2));
    const uint64_t per_block = 256u >> lanes_log2;
    const auto blocks = [&](uint64_t items) { return (items + per_block - 1) / per_block * a.slices; };
    if (blocks(g.n_segments) > 0x7FFFFFFFull) {
        set_error("too many rows and columns for one launch");
        return SDRB_ERR_OVERFLOW;
    }
    if (a.chunk) {
        const uint64_t n_chunks = (g.n_elems + a.chunk - 1) / a.chunk;
        hipLaunchKernelGGL((k_gather_chunks<V, T, Id, WEIGHTED>), dim3((uint32_t)blocks(n_chunks)), dim3(256), 0, stream, a,
                           index, src, n_chunks);
        SDRB_HIP(hipGetLastError());
    }
    const dim3 grid((uint32_t)blocks(g.n_segments));
    if (g.accumulate)
        hipLaunchKernelGGL((k_gather_rows<V, T, O, Id, WEIGHTED, true>), grid, dim3(256), 0, stream, a, index, src, static_cast<O*>(g.out));
    else
        hipLaunchKernelGGL((k_gather_rows<V, T, O, Id, WEIGHTED, false>), grid, dim3(256), 0, stream, a, index, src, static_cast<O*>(g.out));
    SDRB_HIP(hipGetLastError());
    return SDRB_OK;
}

}  // namespace

size_t gather_partial_bytes(uint64_t n_segments, uint64_t n_elems, bool ragged, uint32_t dim) {
    if (n_segments == 0 || n_elems == 0) return 0;
    const uint32_t chunk = chunk_of(n_segments, n_elems);
    if (!ragged && n_elems / n_segments <= chunk) return 0;
    if (n_elems <= chunk) return 0;
    return (size_t)((n_elems + chunk - 1) / chunk) * 2 * dim * sizeof(float);
}

int launch_gather_sum(const GatherSum& g, hipStream_t stream) {
    if (g.n_segments == 0 || g.dim == 0) return SDRB_OK;
    GatherArgs a{};
    a.n_segments = g.n_segments;
    a.n_elems = g.n_elems;
    a.src_rows = g.src_rows;
    a.src_ld = g.src_ld;
    a.out_ld = g.out_ld;
    a.start = g.start;
    a.weight = g.weight;
    a.partials = g.partials;
    a.scale = g.scale;
    a.row_len = g.start ? 0u : (uint32_t)(g.n_elems / g.n_segments);
    a.dim = g.dim;
    a.chunk = g.partials ? chunk_of(g.n_segments, g.n_elems) : 0u;
    return with_type(g.src_type, [&](auto t) {
        return with_type(g.out_type, [&](auto o) {
            using T = decltype(t);
            using O = decltype(o);
            constexpr int V = 16 / sizeof(T);
            const auto go = [&](auto id, auto weighted) {
                using Id = decltype(id);
                constexpr bool W = decltype(weighted)::value;
                return a.dim >= (uint32_t)V ? launch_typed<V, T, O, Id, W>(g, a, stream) : launch_typed<1, T, O, Id, W>(g, a, stream);
            };
            if (g.index_bits == 64) return g.weight ? go(int64_t{}, std::true_type{}) : go(int64_t{}, std::false_type{});
            return g.weight ? go(int32_t{}, std::true_type{}) : go(int32_t{}, std::false_type{});
        });
    });
}

}  // namespace sdrb
