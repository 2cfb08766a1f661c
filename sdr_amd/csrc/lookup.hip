// Ragged gather-sums over a dense matrix: out[s, :] = scale * sum of weight[p] * src[index[p], :] over a segment's
// elements p.  A lookup runs it over the rows of a batch, the table's gradient over the elements sorted by id.
//
// A group of L lanes owns one segment and a slice of the columns, V * SL columns a lane, and adds the segment's elements into
// binary32 registers; the sum is scaled and rounded once to the output's type.  The group's lanes read L elements at a time,
// one each, turn ids into byte offsets, and pass these around by ds_bpermute, so that an element costs its lanes one
// addition, the load, and an fma a column.  Rows of src are read by buffer loads, which yield 0 beyond the matrix: an element
// that contributes nothing has an offset there and a weight of 0, and needs no branch.  (Matrices beyond 2 GiB, or not aligned
// to 4 bytes, are read by address.)
// Short segments (tokens): whole waves, four slices at once, one element a turn: a copy, bound by HBM (16384 tokens of 4096 bf16
// columns in 33-39 us: 245 MB read and written at 6.3 to 7.4 TB/s, some of it from the memory-side cache).
// Long segments (codes): L = 16, two slices of 256 bytes a lane's turn, four elements in flight: bound by L2, and by the issue of vector
// instructions (84 % of the CUs' busy time below; 36 % for fp32 rows of 4004 bytes, which touch a third more lines).  Each XCD (block
// number modulo 8) works through slices of its own, one after another: 512 bytes of every row of a table are what its L2 has
// to hold at a time, not the whole table.  Measured on 4096 rows of 328 of 16384 ids, 1024 bf16 columns (2.75 GB read):
// 114 us = 24 TB/s; slices of 128 bytes 175 us, 256 bytes 128 us, one slice of 1 KiB for all XCDs 226 us.
// S groups share a segment where there are too few of them to fill the chip, and join their sums in LDS.
// A segment of more than `chunk` elements would keep its group busy long after the others: its elements are summed by groups
// that own a chunk of the element list each (k_gather_chunks), and the segment's own group adds those sums up in order.
// Every order of additions follows from the shapes and offsets alone: results repeat bit for bit.
#include <algorithm>

#include "dense_rows.h"

namespace sdrb {

namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kNowhere = 0x80000000u;   // an offset beyond every matrix that is read by buffer loads

struct GatherArgs {
    uint64_t n_segments, n_elems, src_rows, src_ld, out_rows, out_ld;
    const uint32_t* start;
    const uint32_t *keys, *begin, *end;
    const void* index;
    const float* weight;
    float* partials;
    uint32_t row_bytes;      // of src, where it is read by buffer loads
    uint32_t src_bytes;      // its end
    float scale;
    uint32_t row_len;        // where start is null
    uint32_t dim;
    uint32_t chunk;          // longer segments come from `partials` (0: none does)
    uint32_t lanes_log2;     // L
    uint32_t split_log2;     // S
    uint32_t slices;         // of the columns
    uint32_t xcd_slices;     // 1: XCDs take slices one after another
    uint32_t blocks;         // an eighth of a slice's
    uint32_t first_block;    // of the launch
    uint32_t wide_index;     // 64-bit indexes
    uint32_t accumulate;
};

// The elements [lo, hi) of a segment and the row its sum goes to; false where it has none.  Offsets that run backwards or past
// the list are cut to it.
__device__ __forceinline__ bool segment_of(const GatherArgs& a, uint64_t s, uint64_t& lo, uint64_t& hi, uint64_t& row) {
    row = s;
    if (a.keys) {
        row = a.keys[s];
        lo = a.begin[s];
        hi = a.end[s];
        return lo == s && row < a.out_rows;   // the run's first element speaks for it
    }
    if (a.start) {
        lo = a.start[s];
        hi = a.start[s + 1];
        hi = hi < a.n_elems ? hi : a.n_elems;
        lo = lo < hi ? lo : hi;
    } else {
        lo = s * a.row_len;
        hi = lo + a.row_len;
    }
    return true;
}

__device__ __forceinline__ uint32_t from_lane(uint32_t v, uint32_t lane) {
    return (uint32_t)__builtin_amdgcn_ds_bpermute((int)(lane * 4), (int)v);
}

// Where a group stands: its segment (or chunk), its part of the segment, and its lane's columns.  A lane whose columns would run
// past the end reads the last V columns instead and stores only what is its own (from `own`).
// LANES: L where it is known at compile time, else 0
template <int LANES>
__device__ __forceinline__ uint32_t lanes_log2(const GatherArgs& a) {
    if constexpr (LANES == 8) return 3;
    if constexpr (LANES == 16) return 4;
    if constexpr (LANES == 64) return 6;
    return a.lanes_log2;
}
template <int V, int SL, int LANES>
struct Place {
    uint64_t item;
    uint32_t lane, part;
    uint32_t col[SL], own[SL];
    bool live;

    __device__ __forceinline__ Place(const GatherArgs& a, uint32_t slice, uint64_t of) : item(of), live(slice < a.slices) {
        const uint32_t l = lanes_log2<LANES>(a);
        lane = threadIdx.x & ((1u << l) - 1);
        part = (threadIdx.x >> l) & ((1u << a.split_log2) - 1);
#pragma unroll
        for (int j = 0; j < SL; ++j) {
            own[j] = (((slice * SL + j) << l) + lane) * V;
            col[j] = own[j] + V <= a.dim ? own[j] : a.dim - V;
        }
    }
    // of the segments' groups: blocks of one slice each
    __device__ __forceinline__ static Place of_segments(const GatherArgs& a) {
        const uint32_t l = lanes_log2<LANES>(a), items = kThreads >> l >> a.split_log2;   // of a block
        const uint32_t number = a.first_block + blockIdx.x;
        uint32_t slice;
        uint64_t block;
        if (a.xcd_slices) {
            // XCD x takes an eighth of all slices' blocks, slice by slice; of a slice that several share it takes blocks from all over
            const uint32_t unit = (number & 7) * a.slices * a.blocks + (number >> 3), place = unit % (8 * a.blocks);
            slice = unit / (8 * a.blocks);
            block = (uint64_t)(place % a.blocks) * 8 + place / a.blocks;
        } else {
            slice = number % a.slices;
            block = number / a.slices;
        }
        Place p(a, slice, block * items + (threadIdx.x >> l >> a.split_log2));
        p.live = p.live && p.item < a.n_segments;
        return p;
    }
    __device__ __forceinline__ bool stores(const GatherArgs& a, int j) const { return own[j] < a.dim; }
};

using i32x2 = __attribute__((ext_vector_type(2))) int32_t;
using i32x4 = __attribute__((ext_vector_type(4))) int32_t;

// V elements at a byte offset of the matrix; beyond it zeros
template <int V, typename T>
__device__ __forceinline__ void load_at(__amdgpu_buffer_rsrc_t src, uint32_t offset, float (&v)[V]) {
    constexpr int kBytes = V * sizeof(T);
    static_assert(kBytes == 16 || kBytes == 8 || kBytes == 4);
    T t[V];
    if constexpr (kBytes == 16) {
        const i32x4 raw = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(src, (int)offset, 0, 0));
        __builtin_memcpy(t, &raw, sizeof t);
    } else if constexpr (kBytes == 8) {
        const i32x2 raw = __builtin_bit_cast(i32x2, __builtin_amdgcn_raw_buffer_load_b64(src, (int)offset, 0, 0));
        __builtin_memcpy(t, &raw, sizeof t);
    } else {
        const int32_t raw = __builtin_bit_cast(int32_t, __builtin_amdgcn_raw_buffer_load_b32(src, (int)offset, 0, 0));
        __builtin_memcpy(t, &raw, sizeof t);
    }
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = to_f32(t[k]);
}

// acc += the elements [lo, hi) of the list, as far as this part of the segment goes.  U elements a turn (U divides L, or L
// is smaller); the ids of the next L elements are on their way while these are added.
template <int V, int SL, int LANES, int U, bool BUFFER, typename T>
__device__ __forceinline__ void add_elements(const GatherArgs& a, const Place<V, SL, LANES>& at, const T* __restrict__ src, uint64_t lo,
                                             uint64_t hi, float (&acc)[SL][V]) {
    const uint32_t l = lanes_log2<LANES>(a), lanes = 1u << l, first = threadIdx.x & 63 & ~(lanes - 1);   // of the group
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(src), 0, (int)a.src_bytes, 0x00020000);
    const auto id_at = [&](uint64_t p) {
        return a.wide_index ? static_cast<const uint64_t*>(a.index)[p] : (uint64_t)(int64_t) static_cast<const int32_t*>(a.index)[p];
    };
    const uint64_t step = (uint64_t)lanes << a.split_log2;
    uint64_t p = lo + ((uint64_t)at.part << l) + at.lane;
    uint64_t id = p < hi ? id_at(p) : ~0ull;
    float weight = a.weight && p < hi ? a.weight[p] : 1.0f;
    for (uint64_t p0 = p - at.lane; p0 < hi; p0 += step) {
        const bool in = id < a.src_rows;   // (a negative id is a large one)
        const uint32_t offset = in ? (BUFFER ? (uint32_t)id * a.row_bytes : (uint32_t)id) : kNowhere;
        const float w = in ? weight : 0.0f;
        p += step;
        id = p < hi ? id_at(p) : ~0ull;
        if (a.weight) weight = p < hi ? a.weight[p] : 0.0f;
        const uint32_t n = hi - p0 < lanes ? (uint32_t)(hi - p0) : lanes;
        for (uint32_t u = 0; u < n; u += U) {
            float v[U][SL][V], wu[U];
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const bool over = LANES == 0 && U > 1 && u + j >= lanes;   // (a group of fewer lanes than U)
                const uint32_t from = over ? first : first + u + j;
                uint32_t o = from_lane(offset, from);
                wu[j] = __builtin_bit_cast(float, from_lane(__builtin_bit_cast(uint32_t, w), from));
                if (over) {
                    o = kNowhere;
                    wu[j] = 0.0f;
                }
#pragma unroll
                for (int k = 0; k < SL; ++k) {
                    if constexpr (BUFFER) {
                        load_at<V, T>(rsrc, o + at.col[k] * (uint32_t)sizeof(T), v[j][k]);
                    } else {
#pragma unroll
                        for (int c = 0; c < V; ++c) v[j][k][c] = 0.0f;
                        if (o != kNowhere) load_n<V>(src + (uint64_t)o * a.src_ld + at.col[k], v[j][k]);
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < U; ++j)
#pragma unroll
                for (int k = 0; k < SL; ++k)
#pragma unroll
                    for (int c = 0; c < V; ++c) acc[k][c] = fmaf(wu[j], v[j][k][c], acc[k][c]);
        }
    }
}

// The parts' sums, added up in order by the first of them.
template <int V, int SL, int LANES>
__device__ __forceinline__ void join_parts(const GatherArgs& a, uint32_t part, float (&acc)[SL][V], float* shared) {
    const uint32_t parts = 1u << a.split_log2;
    if (parts == 1) return;
#pragma unroll
    for (int k = 0; k < SL; ++k) {
        if (k) __syncthreads();
#pragma unroll
        for (int c = 0; c < V; ++c) shared[c * kThreads + threadIdx.x] = acc[k][c];
        __syncthreads();
        if (part == 0)
            for (uint32_t s = 1; s < parts; ++s)
#pragma unroll
                for (int c = 0; c < V; ++c) acc[k][c] += shared[c * kThreads + threadIdx.x + (s << lanes_log2<LANES>(a))];
    }
}

template <int V, int SL, int LANES, int U, bool BUFFER, typename T, typename O>
__global__ __launch_bounds__(kThreads) void k_gather_rows(GatherArgs a, const T* __restrict__ src, O* __restrict__ out) {
    __shared__ float shared[V * kThreads];
    Place<V, SL, LANES> at = Place<V, SL, LANES>::of_segments(a);
    uint64_t lo = 0, hi = 0, row = 0;
    if (at.live) at.live = segment_of(a, at.item, lo, hi, row);
    if (!at.live) lo = hi = 0;
    float acc[SL][V];
#pragma unroll
    for (int k = 0; k < SL; ++k)
#pragma unroll
        for (int c = 0; c < V; ++c) acc[k][c] = 0.0f;
    if (a.chunk && hi - lo > a.chunk) {
        // chunk c of the element list keeps two sums: of the segment its first element lies in, and of the one its last
        // (some of them on their way at a time: an id of many elements, as words have, would keep its group waiting)
        if (at.part == 0) {
            constexpr int P = V > 4 ? 2 : 4;
            const uint64_t first = lo / a.chunk, last = (hi - 1) / a.chunk;
#pragma unroll
            for (int k = 0; k < SL; ++k)
#pragma unroll 1
                for (uint64_t c0 = first; c0 <= last; c0 += P) {
                    float v[P][V];
#pragma unroll
                    for (int i = 0; i < P; ++i) {
                        const uint64_t c = c0 + i < last ? c0 + i : last;
                        load_n<V>(a.partials + (2 * c + (c * a.chunk < lo ? 1 : 0)) * a.dim + at.col[k], v[i]);
                    }
#pragma unroll
                    for (int i = 0; i < P; ++i)
#pragma unroll
                        for (int j = 0; j < V; ++j) acc[k][j] = c0 + i <= last ? acc[k][j] + v[i][j] : acc[k][j];
                }
        }
    } else {
        add_elements<V, SL, LANES, U, BUFFER>(a, at, src, lo, hi, acc);
    }
    join_parts<V, SL, LANES>(a, at.part, acc, shared);
    if (!at.live || at.part != 0 || (a.accumulate && lo == hi)) return;
#pragma unroll
    for (int k = 0; k < SL; ++k) {
        if (!at.stores(a, k)) break;
        O* to = out + row * a.out_ld + at.col[k];
        if (at.col[k] == at.own[k]) {
            if (a.accumulate) {
                float old[V];
                load_n<V>(to, old);
#pragma unroll
                for (int c = 0; c < V; ++c) acc[k][c] = fmaf(a.scale, acc[k][c], old[c]);
            } else {
#pragma unroll
                for (int c = 0; c < V; ++c) acc[k][c] *= a.scale;
            }
            store_n<V>(to, acc[k]);
        } else {
            const uint32_t skip = at.own[k] - at.col[k];
#pragma unroll
            for (int c = 0; c < V; ++c)
                if ((uint32_t)c >= skip) to[c] = from_f32<O>(a.accumulate ? fmaf(a.scale, acc[k][c], to_f32(to[c])) : acc[k][c] * a.scale);
        }
    }
}

// The sums that chunk c of the element list contributes to segments longer than a chunk.  A block takes a chunk, its groups of 8
// lanes parts of the chunk and as many slices as that leaves, one step after another.  Where no segment is long, it finds
// that and ends: few blocks and few steps of search, since rows of unknown lengths pay for them on every call.
template <int V, int LANES, int U, bool BUFFER, typename T>
__global__ __launch_bounds__(kThreads) void k_gather_chunks(GatherArgs a, const T* __restrict__ src) {
    __shared__ float shared[V * kThreads];
    const uint32_t l = lanes_log2<LANES>(a), group = threadIdx.x >> l, a_step = kThreads >> l >> a.split_log2;   // slices
    const uint64_t c = blockIdx.x;
    const uint64_t c_lo = c * a.chunk, c_hi = c_lo + a.chunk < a.n_elems ? c_lo + a.chunk : a.n_elems;
#pragma unroll 1
    for (int end = 0; end < 2; ++end) {
        const uint64_t p = end ? c_hi - 1 : c_lo;
        uint64_t lo, hi, row;
        if (a.keys) {
            lo = a.begin[p];
            hi = a.keys[p] < a.out_rows ? a.end[p] : lo;
        } else {
            segment_of(a, a.start ? segment_at(a.start, a.n_segments, p) : p / a.row_len, lo, hi, row);
        }
        if (hi - lo <= a.chunk || (end && lo <= c_lo)) continue;   // short, or the first element's segment once more
        for (uint32_t s0 = blockIdx.y * a_step; s0 < a.slices; s0 += gridDim.y * a_step) {
            const Place<V, 1, LANES> at(a, s0 + (group >> a.split_log2), c);
            float acc[1][V];
#pragma unroll
            for (int k = 0; k < V; ++k) acc[0][k] = 0.0f;
            if (at.live) add_elements<V, 1, LANES, U, BUFFER>(a, at, src, lo > c_lo ? lo : c_lo, hi < c_hi ? hi : c_hi, acc);
            join_parts<V, 1, LANES>(a, at.part, acc, shared);
            if (at.part == 0 && at.stores(a, 0)) {
                float* to = a.partials + (2 * c + end) * a.dim + at.col[0];
                if (at.col[0] == at.own[0]) {
                    store_n<V>(to, acc[0]);
                } else {
                    const uint32_t skip = at.own[0] - at.col[0];
#pragma unroll
                    for (int k = 0; k < V; ++k)
                        if ((uint32_t)k >= skip) to[k] = acc[0][k];
                }
            }
            __syncthreads();
        }
    }
}

uint32_t log2_of(uint64_t v) {
    uint32_t l = 0;
    while ((2ull << l) <= v) ++l;
    return l;
}

// lanes of a group: `most`, but no more than the row has vectors
uint32_t group_log2(uint32_t most, uint64_t vectors) { return std::min<uint32_t>(most, log2_of(vectors > 1 ? 2 * vectors - 1 : 1)); }

template <int V, int LANES, bool BUFFER, typename T>
int launch_chunks(const GatherSum& g, GatherArgs a, hipStream_t stream) {
    const uint64_t n_chunks = (g.n_elems + a.chunk - 1) / a.chunk, vectors = (a.dim + V - 1) / V;
    a.lanes_log2 = group_log2(3, vectors);
    const uint32_t groups = kThreads >> a.lanes_log2;
    a.split_log2 = std::min<uint32_t>(log2_of(groups), log2_of(std::max<uint32_t>(a.chunk >> a.lanes_log2, 1)));
    a.slices = (uint32_t)((vectors + (1u << a.lanes_log2) - 1) >> a.lanes_log2);
    while (a.split_log2 > 2 && (groups >> a.split_log2) < a.slices) --a.split_log2;
    // Slices side by side: four where one load tells whether a run is long, and as many as the chip has room for where chunks are few,
    // since long segments wait for the slowest chunk (4060 tokens of 692 ids, 896 fp32 columns: 5.9 us, 13.8 with one)
    const uint32_t steps = (a.slices + (groups >> a.split_log2) - 1) / (groups >> a.split_log2);
    const uint32_t across = std::min(steps, std::max<uint32_t>(g.keys ? 4 : 1, (uint32_t)(512 / n_chunks)));
    hipLaunchKernelGGL((k_gather_chunks<V, LANES, 8, BUFFER, T>), dim3((uint32_t)n_chunks, across), dim3(kThreads), 0,
                       stream, a, static_cast<const T*>(g.src));
    SDRB_HIP(hipGetLastError());
    return SDRB_OK;
}

template <int V, int SL, int LANES, int U, bool BUFFER, typename T, typename O>
int launch_rows(const GatherSum& g, GatherArgs a, uint64_t mean, hipStream_t stream) {
    const uint64_t vectors = (a.dim + V - 1) / V;
    a.lanes_log2 = LANES ? log2_of(LANES) : group_log2(U == 1 ? 6 : 4, vectors);
    const uint64_t a_slice = (uint64_t)SL << a.lanes_log2;
    a.slices = (uint32_t)((vectors + a_slice - 1) / a_slice);
    // S: waves for the whole chip, eight a SIMD, as long as every part has elements to add
    const uint64_t groups = g.n_segments * a.slices, enough = (uint64_t)1024 * 8 * (64u >> a.lanes_log2);
    a.split_log2 = 0;
    while ((kThreads >> a.lanes_log2 >> a.split_log2) > 1 && (groups << a.split_log2) < enough && (1ull << a.split_log2) << a.lanes_log2 < mean)
        ++a.split_log2;
    const uint64_t per_block = kThreads >> a.lanes_log2 >> a.split_log2, blocks = (g.n_segments + per_block - 1) / per_block;
    a.xcd_slices = U > 1 && LANES != 64 && blocks >= 8;
    a.blocks = (uint32_t)((blocks + 7) / 8);
    const uint64_t grid = (a.xcd_slices ? 8ull * a.blocks : blocks) * a.slices;
    if (grid > 0x7FFFFFFFull) {
        set_error("too many rows and columns for one launch");
        return SDRB_ERR_OVERFLOW;
    }
    return in_launches(grid, kThreads, [&](uint64_t first, uint32_t n_blocks) {
        a.first_block = (uint32_t)first;
        hipLaunchKernelGGL((k_gather_rows<V, SL, LANES, U, BUFFER, T, O>), dim3(n_blocks), dim3(kThreads), 0, stream, a,
                           static_cast<const T*>(g.src), static_cast<O*>(g.out));
        SDRB_HIP(hipGetLastError());
        return SDRB_OK;
    });
}

// elements to reckon with in a segment: without chunks one of ragged segments may hold them all
uint64_t mean_of(const GatherSum& g) { return g.start && !g.chunk ? g.n_elems : g.n_elems / g.n_segments; }

template <bool BUFFER, typename T, typename O>
int launch_typed(const GatherSum& g, GatherArgs a, hipStream_t stream) {
    // long segments read more than they write: 16 bytes a load; short ones: 16 bytes at most a load or store
    constexpr int kWide = 16 / sizeof(T), kEven = 16 / (sizeof(T) > sizeof(O) ? sizeof(T) : sizeof(O));
    const uint64_t mean = mean_of(g);
    if (a.chunk) {
        const int rc = a.dim >= 8u * kWide ? launch_chunks<kWide, 8, BUFFER, T>(g, a, stream) : launch_chunks<kWide, 0, BUFFER, T>(g, a, stream);
        if (rc != SDRB_OK) return rc;
    }
    if (mean >= 3) {
        // Slices of 512 bytes, two of 256 a lane's turn, from four of them on, unless they leave a tenth more lanes without columns:
        // 8192 rows of 40 of 4096 ids, 1024 bf16 columns 32.4 us (slices of 256 bytes: 34.2), 512 columns 20.3 (17.3)
        const uint32_t vectors = (a.dim + kWide - 1) / kWide, twos = (vectors + 31) / 32 * 32, ones = (vectors + 15) / 16 * 16;
        if (vectors >= 128 && 10 * twos <= 11 * ones) return launch_rows<kWide, 2, 16, 4, BUFFER, T, O>(g, a, mean, stream);
        if (a.dim >= 16u * kWide) return launch_rows<kWide, 1, 16, 8, BUFFER, T, O>(g, a, mean, stream);
        return launch_rows<kWide, 1, 0, 4, BUFFER, T, O>(g, a, mean, stream);
    }
    if (a.dim >= 64u * kEven) {
        if (g.keys) return launch_rows<kEven, 4, 64, 2, BUFFER, T, O>(g, a, mean, stream);   // (runs have an element at least)
        return launch_rows<kEven, 4, 64, 1, BUFFER, T, O>(g, a, mean, stream);
    }
    return launch_rows<kEven, 1, 0, 1, BUFFER, T, O>(g, a, mean, stream);
}

}  // namespace

// The longest run of elements that one group of lanes sums by itself: long enough that few segments need a second step, short
// enough that the longest does not outlast the rest; 4096 of them if that leaves 1024 elements or fewer, since all have to be looked
// at (a million elements of 65536 ids, none of whose segments is long: 13 us, and 45 with chunks of 64).
// None for a few thousand elements in few enough segments and columns that a whole block can share each: one launch, and no scratch.
// (2000 elements in 200 rows of 512 columns 5.0 us against 6.4, 12.6 against 13.6 with all of them in one row; in 200 rows of 2048
// columns 10.4 against 7.1, so not there.)
uint32_t segment_chunk(uint64_t n_segments, uint64_t n_elems, uint32_t dim, bool ragged) {
    if (n_segments == 0 || n_elems == 0) return 0;
    const uint64_t mean = n_elems / n_segments;
    if (mean >= 3 && n_elems <= 4096 && n_segments * dim <= 1u << 18) return 0;
    uint32_t chunk = 64;
    while (((chunk < 4 * mean || n_elems > 4096ull * chunk) && chunk < 1024) || n_elems > ((uint64_t)chunk << 22)) chunk *= 2;   // (one launch: 4 million at most)
    return n_elems <= chunk || (!ragged && mean <= chunk) ? 0 : chunk;
}
// The same for runs of a sorted list, most of them of an element or two.  Words' frequencies make the longest run a sixteenth of
// the list: short chunks leave its group many sums to add up, long ones many elements.  Measured with chunks of 16, 32, 64, 128 and
// 256: 4000 elements of 512 columns 27.4, 25.9, 32, 39 and 52 us; 60000 of 1024 187, 152, 137, 154 and 201; 262144 of 512 260,
// 260, 260, 247 and 258.
uint32_t run_chunk(uint64_t n_elems) {
    uint32_t chunk = n_elems <= 1024 ? 16 : 32;
    while (n_elems > (chunk < 128 ? 1024ull : 4096ull) * chunk) chunk *= 2;
    return n_elems <= 64 ? 0 : chunk;
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
    a.index = g.index;
    a.wide_index = g.index_bits == 64;
    a.weight = g.weight;
    a.partials = g.partials;
    a.scale = g.scale;
    a.row_len = g.start ? 0u : (uint32_t)(g.n_elems / g.n_segments);
    a.dim = g.dim;
    a.keys = g.keys;
    a.begin = g.begin;
    a.end = g.end;
    a.out_rows = g.out_rows;
    a.chunk = g.chunk;
    a.accumulate = g.accumulate ? 1u : 0u;
    return with_type(g.src_type, [&](auto t) {
        return with_type(g.out_type, [&](auto o) {
            using T = decltype(t);
            using O = decltype(o);
            constexpr uint32_t kWide = 16 / sizeof(T);
            const uint64_t bytes = g.src_rows ? ((g.src_rows - 1) * g.src_ld + a.dim) * sizeof(T) : 0;
            const bool by_words = reinterpret_cast<uintptr_t>(g.src) % 4 == 0 && g.src_ld * sizeof(T) % 4 == 0 && a.dim * sizeof(T) % 4 == 0;
            if (a.dim < kWide) {   // narrower than a load: a column a lane
                if (a.chunk)
                    if (const int rc = launch_chunks<1, 0, false, T>(g, a, stream)) return rc;
                return launch_rows<1, 1, 0, 1, false, T, O>(g, a, mean_of(g), stream);
            }
            if (bytes >= kNowhere || !by_words) return launch_typed<false, T, O>(g, a, stream);
            a.row_bytes = (uint32_t)(g.src_ld * sizeof(T));
            a.src_bytes = (uint32_t)bytes;
            return launch_typed<true, T, O>(g, a, stream);
        });
    });
}

}  // namespace sdrb
