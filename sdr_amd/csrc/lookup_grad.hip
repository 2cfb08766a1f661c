// Gradients of a lookup out[r, :] = scale * sum over row r's elements e of w[e] * table[id[e], :].
//
// To the table: d table[v, :] = scale * sum over the elements e with id[e] = v of w[e] * d out[row(e), :].  The elements are
// sorted by id -- a stable radix sort, so that the elements of one id keep their order -- and the sums run over the
// sorted list like a lookup whose rows are the ids (lookup.hip): no atomic addition, the same bits every time, and the
// work of an id that many rows hold is shared out.
// To the weights: d w[e] = scale * <d out[row(e), :], table[id[e], :]>, a dot product an element.
#include <algorithm>

#include "dense_rows.h"

namespace sdrb {

namespace {

// ---- sorting elements by id ---------------------------------------------------------------------------------------------
// Keys are ids, or n_table_rows for an element that contributes nothing (an id outside the table, or an element that no row
// holds), so they take bits(n_table_rows).  A pass sorts by a digit of them, stably: the 64 elements of a wave's turn find
// the others of their digit by a ballot a digit bit, and a wave counts in LDS what its earlier turns have seen of each digit.
//
// Up to 16384 elements one block does it all in LDS (k_sort_small), 8 bits a pass, the elements in registers between passes:
// every further launch costs more than a pass.  More elements take three launches a pass: digits counted by tile, the
// counts summed over tiles, and the elements sent to their places.  Digits have up to 12 bits there, so that ids below
// 4096 -- the widths of sparse codes -- need one pass, and then the counts are the segments' starts too.

struct SortArgs {
    const void* ids;
    const uint32_t* off;     // row offsets, or null: rows of row_len
    const float* weight;     // or null
    uint64_t n, n_keys, n_rows;
    uint32_t row_len, wide;  // wide: 64-bit ids
    uint32_t key_bits;
};

__device__ __forceinline__ uint32_t key_of(const SortArgs& a, uint64_t e) {
    const uint64_t id = a.wide ? static_cast<const uint64_t*>(a.ids)[e] : (uint64_t)(int64_t) static_cast<const int32_t*>(a.ids)[e];
    const bool in = id < a.n_keys && (!a.off || (e >= a.off[0] && e < a.off[a.n_rows]));   // (a negative id is a large one)
    return in ? (uint32_t)id : (uint32_t)a.n_keys;
}
// the row of element e
__device__ __forceinline__ uint32_t row_of(const uint32_t* __restrict__ off, uint64_t n_rows, uint32_t row_len, uint64_t e) {
    if (!off) return (uint32_t)e / row_len;
    uint64_t lo = 0, hi = n_rows;   // last row that starts at or before e
    while (hi - lo > 1) {
        const uint64_t mid = (lo + hi) >> 1;
        if (off[mid] <= e) lo = mid;
        else hi = mid;
    }
    return (uint32_t)lo;
}
__device__ __forceinline__ uint32_t lanes_below(unsigned long long mask) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u));
}
// the lanes of the wave that hold the same digit, of those that are live
template <int BITS>
__device__ __forceinline__ unsigned long long same_digit(uint32_t digit, bool live) {
    const unsigned long long on = __builtin_amdgcn_ballot_w64(live);
    uint32_t lo = (uint32_t)on, hi = (uint32_t)(on >> 32);
#pragma unroll
    for (int b = 0; b < BITS; ++b) {
        const uint32_t set = (uint32_t)((int32_t)(digit << (31 - b)) >> 31);   // all ones or none
        const unsigned long long with = __builtin_amdgcn_ballot_w64(set != 0);
        lo &= ~((uint32_t)with ^ set);
        hi &= ~((uint32_t)(with >> 32) ^ set);
    }
    return ((unsigned long long)hi << 32) | lo;
}
// Of equal digits, what the wave's earlier turns and the lower lanes hold; counter[digit] goes up by this turn's.
template <int BITS>
__device__ __forceinline__ uint32_t rank_in_wave(uint32_t* counter, uint32_t digit, bool live) {
    const unsigned long long same = same_digit<BITS>(digit, live);
    const uint32_t below = lanes_below(same);
    uint32_t before = 0;
    if (live) before = counter[digit];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // all have read before the first of them writes
    __builtin_amdgcn_wave_barrier();
    if (live && below == 0) counter[digit] = before + (uint32_t)__builtin_popcountll(same);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    return before + below;
}
constexpr uint32_t kSmall = 16384, kSmallThreads = 1024, kSmallWaves = kSmallThreads / 64, kSmallTurns = kSmall / kSmallThreads;
constexpr uint64_t kStartsInSort = 4096;   // up to so many keys the one block finds their starts as well, four a thread

__global__ __launch_bounds__(kSmallThreads) void k_sort_small(SortArgs a, uint32_t* __restrict__ keys_out, int32_t* __restrict__ row_out,
                                                              float* __restrict__ weight_out, uint32_t* __restrict__ start) {
    __shared__ uint32_t key_at[kSmall];
    __shared__ uint16_t elem_at[kSmall];
    __shared__ uint32_t counter[kSmallWaves][256];
    __shared__ uint32_t digit_waves[4];
    const uint32_t n = (uint32_t)a.n, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t turns = (n + kSmallThreads - 1) / kSmallThreads;   // a wave owns turns * 64 neighbouring elements
    uint32_t key[kSmallTurns], elem[kSmallTurns], place[kSmallTurns];
#pragma unroll
    for (uint32_t t = 0; t < kSmallTurns; ++t) {
        elem[t] = (wave * turns + t) * 64 + lane;
        key[t] = t < turns && elem[t] < n ? key_of(a, elem[t]) : 0u;
    }
    for (uint32_t shift = 0; shift < a.key_bits; shift += 8) {
        for (uint32_t k = threadIdx.x; k < kSmallWaves * 256; k += kSmallThreads) counter[k >> 8][k & 255] = 0;
        __syncthreads();
#pragma unroll
        for (uint32_t t = 0; t < kSmallTurns; ++t) {
            if (t >= turns) continue;
            // (positions, not elements, say which lanes are live: after the first pass the last ones are the largest keys)
            const bool live = (wave * turns + t) * 64 + lane < n;
            place[t] = rank_in_wave<8>(counter[wave], (key[t] >> shift) & 255u, live);
        }
        __syncthreads();
        if (threadIdx.x < 256) {   // a digit a thread: sums over the waves, then over the digits
            uint32_t total = 0;
            for (uint32_t w = 0; w < kSmallWaves; ++w) {
                const uint32_t here = counter[w][threadIdx.x];
                counter[w][threadIdx.x] = total;
                total += here;
            }
            const uint32_t sum = scan_lanes<64>(total);
            if (lane == 63) digit_waves[wave] = sum;
            key_at[threadIdx.x] = sum - total;   // (its contents have been read)
        }
        __syncthreads();
        if (threadIdx.x < 256) {
            uint32_t before = key_at[threadIdx.x];
            for (uint32_t w = 0; w < wave; ++w) before += digit_waves[w];
            for (uint32_t w = 0; w < kSmallWaves; ++w) counter[w][threadIdx.x] += before;
        }
        __syncthreads();
#pragma unroll
        for (uint32_t t = 0; t < kSmallTurns; ++t) {
            if (t >= turns) continue;
            if ((wave * turns + t) * 64 + lane < n) {
                const uint32_t to = counter[wave][(key[t] >> shift) & 255u] + place[t];
                key_at[to] = key[t];
                elem_at[to] = (uint16_t)elem[t];
            }
        }
        __syncthreads();
#pragma unroll
        for (uint32_t t = 0; t < kSmallTurns; ++t) {
            if (t >= turns) continue;
            const uint32_t p = (wave * turns + t) * 64 + lane;
            if (p < n) {
                key[t] = key_at[p];
                elem[t] = elem_at[p];
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (uint32_t t = 0; t < kSmallTurns; ++t) {
        if (t >= turns) continue;
        const uint32_t p = (wave * turns + t) * 64 + lane;
        if (p < n) {
            keys_out[p] = key[t];
            row_out[p] = (int32_t)row_of(a.off, a.n_rows, a.row_len, elem[t]);
            if (a.weight) weight_out[p] = a.weight[elem[t]];
            key_at[p] = key[t];
        }
    }
    if (a.n_keys > kStartsInSort) return;
    __syncthreads();
    for (uint32_t v = threadIdx.x; v <= a.n_keys; v += kSmallThreads) {
        uint32_t lo = 0, hi = n;
        while (lo < hi) {
            const uint32_t mid = (lo + hi) >> 1;
            if (key_at[mid] < v) lo = mid + 1;
            else hi = mid;
        }
        start[v] = lo;
    }
}

constexpr uint32_t kTileWaves = 4, kMostDigits = 4096;   // of a tile of the sort of many elements

struct PassArgs {
    const uint32_t* keys;    // null in the first pass: the ids themselves
    const uint32_t* elems;
    uint32_t* counts;        // [tile][digit]
    uint32_t* totals;        // [digit]
    uint32_t shift, bits, turns, n_tiles;   // turns: of 64 elements a wave
    uint32_t last;
    uint32_t* keys_out;
    uint32_t* elems_out;
    int32_t* row_out;        // in the last pass
    float* weight_out;
    uint32_t* start;         // in the only pass
};
__device__ __forceinline__ uint32_t pass_key(const SortArgs& a, const PassArgs& s, uint64_t p) { return s.keys ? s.keys[p] : key_of(a, p); }

__global__ __launch_bounds__(256) void k_count(SortArgs a, PassArgs s) {
    __shared__ uint32_t h[kMostDigits];
    const uint32_t digits = 1u << s.bits;
    for (uint32_t d = threadIdx.x; d < digits; d += 256) h[d] = 0;
    __syncthreads();
    const uint64_t tile = (uint64_t)kTileWaves * s.turns * 64, t0 = blockIdx.x * tile;
    for (uint64_t i = threadIdx.x; i < tile && t0 + i < a.n; i += 256)
        atomicAdd(&h[(pass_key(a, s, t0 + i) >> s.shift) & (digits - 1)], 1u);   // (a count does not depend on their order)
    __syncthreads();
    for (uint32_t d = threadIdx.x; d < digits; d += 256) s.counts[(uint64_t)blockIdx.x * digits + d] = h[d];
}

// counts[tile][digit] become what the tiles before hold of the digit; totals[digit] what all do
__global__ __launch_bounds__(64) void k_sum_tiles(PassArgs s) {
    const uint32_t digits = 1u << s.bits, d = blockIdx.x * 64 + threadIdx.x;
    if (d >= digits) return;
    uint32_t total = 0;
    uint32_t* at = s.counts + d;
    constexpr uint32_t kAhead = 32;   // reads in flight
    for (uint32_t t = 0; t < s.n_tiles; t += kAhead) {
        uint32_t c[kAhead];
#pragma unroll
        for (uint32_t k = 0; k < kAhead; ++k) c[k] = t + k < s.n_tiles ? at[(uint64_t)(t + k) * digits] : 0u;
#pragma unroll
        for (uint32_t k = 0; k < kAhead; ++k) {
            if (t + k < s.n_tiles) at[(uint64_t)(t + k) * digits] = total;
            total += c[k];
        }
    }
    s.totals[d] = total;
}

template <int BITS>
__global__ __launch_bounds__(256) void k_scatter(SortArgs a, PassArgs s) {
    constexpr uint32_t kDigits = 1u << BITS, kEach = (kDigits + 255) / 256;   // digits of a thread
    __shared__ uint32_t next[kTileWaves][kDigits];
    __shared__ uint32_t sums[kEach * 4];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t total[kEach], tiles_before[kEach];
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) {   // on their way while the tile's own digits are counted
        const uint32_t d = i * 256 + threadIdx.x;
        total[i] = d < kDigits ? s.totals[d] : 0u;
        tiles_before[i] = d < kDigits ? s.counts[(uint64_t)blockIdx.x * kDigits + d] : 0u;
    }
    for (uint32_t k = threadIdx.x; k < kTileWaves * kDigits; k += 256) next[k >> BITS][k & (kDigits - 1)] = 0;
    __syncthreads();
    const uint64_t w0 = ((uint64_t)blockIdx.x * kTileWaves + wave) * s.turns * 64;
    for (uint32_t t = 0; t < s.turns; ++t) {
        const uint64_t p = w0 + t * 64 + lane;
        if (p < a.n) atomicAdd(&next[wave][(pass_key(a, s, p) >> s.shift) & (kDigits - 1)], 1u);
    }
    // a digit's first place: the digits before it, the tiles before this one, the waves before
    uint32_t first[kEach];
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) {
        const uint32_t sum = scan_lanes<64>(total[i]);
        if (lane == 63) sums[i * 4 + wave] = sum;
        first[i] = sum - total[i];
    }
    __syncthreads();
    if (wave == 0) {   // the sums of 64 digits each, at most 64 of them
        const uint32_t here = lane < kEach * 4 ? sums[lane] : 0u, sum = scan_lanes<64>(here);
        if (lane < kEach * 4) sums[lane] = sum - here;
    }
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) {
        const uint32_t d = i * 256 + threadIdx.x;
        if (d >= kDigits) continue;
        first[i] += sums[i * 4 + wave];
        if (s.start && blockIdx.x == 0 && d <= a.n_keys) s.start[d] = first[i];
        uint32_t at = first[i] + tiles_before[i];
#pragma unroll
        for (uint32_t w = 0; w < kTileWaves; ++w) {
            const uint32_t here = next[w][d];
            next[w][d] = at;
            at += here;
        }
    }
    __syncthreads();
    for (uint32_t t = 0; t < s.turns; ++t) {
        const uint64_t p = w0 + t * 64 + lane;
        const bool live = p < a.n;
        const uint32_t key = live ? pass_key(a, s, p) : 0u;
        const uint32_t to = rank_in_wave<BITS>(next[wave], (key >> s.shift) & (kDigits - 1), live);
        if (!live) continue;
        const uint32_t e = s.elems ? s.elems[p] : (uint32_t)p;
        if (s.last) {
            s.row_out[to] = (int32_t)row_of(a.off, a.n_rows, a.row_len, e);
            if (a.weight) s.weight_out[to] = a.weight[e];
        } else {
            s.elems_out[to] = e;
        }
        if (s.keys_out) s.keys_out[to] = key;
    }
}

// start[v] = the first sorted position whose key is >= v, for v in [0, n_keys]
__global__ __launch_bounds__(256) void k_starts(const uint32_t* __restrict__ keys, uint64_t n, uint64_t n_keys,
                                                uint32_t* __restrict__ start) {
    const uint64_t v = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (v > n_keys) return;
    uint64_t lo = 0, hi = n;
    while (lo < hi) {
        const uint64_t mid = (lo + hi) >> 1;
        if (keys[mid] < v) lo = mid + 1;
        else hi = mid;
    }
    start[v] = (uint32_t)lo;
}

// ---- the gradient to the weights ------------------------------------------------------------------------------------------
// A wave takes 64 elements, a lane finding the row and the table row of each, and works through them B at a time: every lane
// loads 16 bytes of the B rows of grad and table, column after column, and the B sums over the lanes are formed together: in
// three steps eight values a lane become one value an eighth of the lanes, half of the values changing sides each time.
template <typename T, typename G>
__global__ __launch_bounds__(256) void k_weight_grad(SortArgs a, const G* __restrict__ grad, uint64_t grad_ld, const T* __restrict__ table,
                                                     uint64_t table_ld, uint32_t dim, float scale, float* __restrict__ out) {
    constexpr int V = 16 / (sizeof(T) > sizeof(G) ? sizeof(T) : sizeof(G)), B = 8;
    const uint64_t e0 = ((uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * 64;
    const uint32_t lane = threadIdx.x & 63;
    if (e0 >= a.n) return;
    uint32_t id = (uint32_t)a.n_keys, row = 0;
    if (e0 + lane < a.n) {
        id = key_of(a, e0 + lane);
        row = row_of(a.off, a.n_rows, a.row_len, e0 + lane);
    }
    float mine = 0.0f;   // of the lane's own element
    const uint32_t n = a.n - e0 < 64 ? (uint32_t)(a.n - e0) : 64;
    for (uint32_t u = 0; u < n; u += B) {
        float sum[B];
        const T* t[B];
        const G* g[B];
        uint32_t live = 0;
#pragma unroll
        for (int j = 0; j < B; ++j) {
            const uint32_t of_id = (uint32_t)__builtin_amdgcn_readlane((int)id, (int)(u + j)), of_row = (uint32_t)__builtin_amdgcn_readlane((int)row, (int)(u + j));
            if (of_id < a.n_keys) live |= 1u << j;
            t[j] = table + (uint64_t)(of_id < a.n_keys ? of_id : 0u) * table_ld;
            g[j] = grad + (uint64_t)of_row * grad_ld;
            sum[j] = 0.0f;
        }
        if (live == 0) continue;
        const bool one_row = g[0] == g[1] && g[0] == g[2] && g[0] == g[3] && g[0] == g[4] && g[0] == g[5] && g[0] == g[6] && g[0] == g[7];
        for (uint32_t c = lane * V; c < dim; c += 64 * V) {
            if (c + V <= dim) {
                float x[B][V], y[B][V];
#pragma unroll
                for (int j = 0; j < B; ++j) load_n<V>(t[j] + c, x[j]);
                if (one_row) {
                    load_n<V>(g[0] + c, y[0]);
#pragma unroll
                    for (int j = 0; j < B; ++j)
#pragma unroll
                        for (int k = 0; k < V; ++k) sum[j] = fmaf(x[j][k], y[0][k], sum[j]);
                } else {
#pragma unroll
                    for (int j = 0; j < B; ++j) load_n<V>(g[j] + c, y[j]);
#pragma unroll
                    for (int j = 0; j < B; ++j)
#pragma unroll
                        for (int k = 0; k < V; ++k) sum[j] = fmaf(x[j][k], y[j][k], sum[j]);
                }
            } else {
                for (uint32_t k = c; k < dim; ++k)
#pragma unroll
                    for (int j = 0; j < B; ++j) sum[j] = fmaf(to_f32(t[j][k]), to_f32(g[j][k]), sum[j]);
            }
        }
        // lane bits 0, 1, 2 choose which half of the values a lane keeps; what is left is that of element lane & 7
        const auto halve = [&](auto count, int bit) {
            constexpr int kHalf = decltype(count)::value / 2;
            const bool high = (lane >> bit) & 1u;
#pragma unroll
            for (int j = 0; j < kHalf; ++j) {
                const float keep = high ? sum[2 * j + 1] : sum[2 * j], give = high ? sum[2 * j] : sum[2 * j + 1];
                sum[j] = keep + __shfl_xor(give, 1 << bit, 64);
            }
        };
        halve(std::integral_constant<int, 8>{}, 0);
        halve(std::integral_constant<int, 4>{}, 1);
        halve(std::integral_constant<int, 2>{}, 2);
#pragma unroll
        for (int s = 8; s < 64; s <<= 1) sum[0] += __shfl_xor(sum[0], s, 64);
        if (lane >= u && lane < u + B && ((live >> (lane - u)) & 1u)) mine = scale * sum[0];   // (u is a multiple of 8)
    }
    if (e0 + lane < a.n) out[e0 + lane] = mine;
}

size_t up(size_t bytes) { return (bytes + 255) / 256 * 256; }

uint32_t bits_of(uint64_t v) {
    uint32_t b = 1;
    while (v >> b) ++b;
    return b;
}

// How many elements are sorted by more than one block: turns of 64 a wave, so that the tiles are some 500 at most, and passes.
struct Passes {
    uint32_t turns, n_tiles, count, bits;
    Passes(uint64_t n, uint32_t key_bits) {
        turns = 8;
        while (turns < 64 && n > (uint64_t)512 * kTileWaves * turns * 64) turns *= 2;
        n_tiles = (uint32_t)((n + kTileWaves * turns * 64 - 1) / (kTileWaves * turns * 64));
        count = (key_bits + 11) / 12;
        bits = std::max((key_bits + count - 1) / count, 8u);
    }
};

SortArgs sort_args(const sdrb_rows& rows, uint64_t n_table_rows) {
    SortArgs a{};
    a.ids = rows.ids;
    a.off = rows.row_offsets;
    a.weight = rows.weights;
    a.n = rows.n_elems;
    a.n_keys = n_table_rows;
    a.n_rows = rows.n_rows;
    a.row_len = rows.row_offsets || !rows.n_rows ? 1u : (uint32_t)(rows.n_elems / rows.n_rows);
    a.wide = rows.id_bits == 64;
    a.key_bits = bits_of(n_table_rows);
    return a;
}

// what a sort and the sums after it keep in the caller's scratch
struct Scratch {
    uint32_t *keys[2], *elems[2], *counts, *totals, *start;
    int32_t* row;
    float* weight;
    float* partials;
    size_t bytes;
    Scratch(void* base, uint64_t n, uint64_t n_keys, bool weighted, uint32_t dim) {
        size_t at = 0;
        const auto take = [&](size_t count) {
            char* p = static_cast<char*>(base) + (base ? at : 0);
            at += up(count * 4);
            return reinterpret_cast<uint32_t*>(p);
        };
        const Passes p(n, bits_of(n_keys));
        const bool small = n <= kSmall;
        row = reinterpret_cast<int32_t*>(take(n));
        weight = reinterpret_cast<float*>(take(weighted ? n : 0));
        for (int k = 0; k < 2; ++k) {   // as many as the passes write: k_starts reads the keys of more than one
            keys[k] = take(small ? (k ? 0 : n) : p.count > 1 ? n : 0);
            elems[k] = take(!small && p.count > 1u + k ? n : 0);
        }
        counts = take(small ? 0 : (size_t)p.n_tiles << p.bits);
        totals = take(small ? 0 : (size_t)1 << p.bits);
        start = take(n_keys + 1);
        partials = gather_partial_bytes(n_keys, n, true, dim) ? reinterpret_cast<float*>(take(0)) : nullptr;
        bytes = at + gather_partial_bytes(n_keys, n, true, dim);
    }
};

int sort_by_id(const SortArgs& a, const Scratch& s, hipStream_t stream) {
    const uint32_t* sorted = nullptr;   // keys whose starts are still to be found
    if (a.n <= kSmall) {
        hipLaunchKernelGGL(k_sort_small, dim3(1), dim3(kSmallThreads), 0, stream, a, s.keys[0], s.row, s.weight, s.start);
        SDRB_HIP(hipGetLastError());
        if (a.n_keys > kStartsInSort) sorted = s.keys[0];
    } else {
        const Passes passes(a.n, a.key_bits);
        for (uint32_t k = 0; k < passes.count; ++k) {
            PassArgs p{};
            p.keys = k ? s.keys[(k - 1) & 1] : nullptr;
            p.elems = k ? s.elems[(k - 1) & 1] : nullptr;
            p.counts = s.counts;
            p.totals = s.totals;
            p.shift = k * passes.bits;
            p.bits = passes.bits;
            p.turns = passes.turns;
            p.n_tiles = passes.n_tiles;
            p.last = k + 1 == passes.count;
            p.keys_out = passes.count > 1 ? s.keys[k & 1] : nullptr;
            p.elems_out = p.last ? nullptr : s.elems[k & 1];
            p.row_out = s.row;
            p.weight_out = s.weight;
            p.start = passes.count == 1 ? s.start : nullptr;
            hipLaunchKernelGGL(k_count, dim3(passes.n_tiles), dim3(256), 0, stream, a, p);
            SDRB_HIP(hipGetLastError());
            hipLaunchKernelGGL(k_sum_tiles, dim3(((1u << passes.bits) + 63) / 64), dim3(64), 0, stream, p);
            SDRB_HIP(hipGetLastError());
            const auto scatter = passes.bits == 12 ? &k_scatter<12> : passes.bits == 11 ? &k_scatter<11> : passes.bits == 10 ? &k_scatter<10> : passes.bits == 9 ? &k_scatter<9> : &k_scatter<8>;
            hipLaunchKernelGGL(scatter, dim3(passes.n_tiles), dim3(256), 0, stream, a, p);
            SDRB_HIP(hipGetLastError());
        }
        if (passes.count > 1) sorted = s.keys[(passes.count - 1) & 1];
    }
    if (sorted) {
        hipLaunchKernelGGL(k_starts, dim3((uint32_t)(a.n_keys / 256 + 1)), dim3(256), 0, stream, sorted, a.n, a.n_keys, s.start);
        SDRB_HIP(hipGetLastError());
    }
    return SDRB_OK;
}

}  // namespace

size_t table_grad_scratch_bytes(uint64_t n_elems, uint64_t n_table_rows, bool weighted, uint32_t dim) {
    return Scratch(nullptr, n_elems, n_table_rows, weighted, dim).bytes;
}

int launch_table_grad(int device, const sdrb_rows& rows, const sdrb_dense& grad, float scale, bool accumulate, const sdrb_dense& out,
                      void* scratch, hipStream_t stream) {
    const uint32_t dim = (uint32_t)out.n_cols;
    const Scratch s(scratch, rows.n_elems, out.n_rows, rows.weights != nullptr, dim);
    const SortArgs a = sort_args(rows, out.n_rows);
    if (const int rc = sort_by_id(a, s, stream)) return rc;
    GatherSum g{};
    g.device = device;
    g.n_segments = out.n_rows;
    g.n_elems = rows.n_elems;
    g.start = s.start;
    g.index = s.row;
    g.index_bits = 32;
    g.weight = rows.weights ? s.weight : nullptr;
    g.src = grad.data;
    g.src_type = grad.type;
    g.src_rows = grad.n_rows;
    g.src_ld = grad.ld;
    g.dim = dim;
    g.out = out.data;
    g.out_type = out.type;
    g.out_ld = out.ld;
    g.scale = scale;
    g.accumulate = accumulate;
    g.partials = s.partials;
    return launch_gather_sum(g, stream);
}

int launch_weight_grad(const sdrb_rows& rows, const sdrb_dense& grad, const sdrb_dense& table, float scale, float* out,
                       hipStream_t stream) {
    if (rows.n_elems == 0) return SDRB_OK;
    const SortArgs a = sort_args(rows, table.n_rows);
    return with_type(table.type, [&](auto t) {
        return with_type(grad.type, [&](auto g) {
            using T = decltype(t);
            using G = decltype(g);
            hipLaunchKernelGGL((k_weight_grad<T, G>), dim3((uint32_t)((a.n + 255) / 256)), dim3(256), 0, stream, a,
                               static_cast<const G*>(grad.data), grad.ld, static_cast<const T*>(table.data), table.ld, (uint32_t)table.n_cols,
                               scale, out);
            SDRB_HIP(hipGetLastError());
            return SDRB_OK;
        });
    });
}

}  // namespace sdrb
