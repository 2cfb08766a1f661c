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
// Few elements one block sorts all by itself in LDS (k_sort_small), 9 bits a pass, in registers between passes: one launch, and
// its time grows with them, since a block has one CU's issue.  More elements take three launches a pass: digits counted by tile, the
// counts summed over tiles, and the elements sent to their places.  Digits have up to 12 bits there, so that ids below
// 4096 -- the widths of sparse codes -- need one pass, and then the counts are the segments' starts too.
// Measured: up to 1024 elements 6 us, 4096 14, 16384 42, in one block (bound by its issue: some 150 instructions a turn of 64);
// 327680 elements of 2048 ids 4 us to count, 7 to sum and 14 to send; 1.3 million of 16384 ids, two passes, 7, 6 and 27, then 7, 6
// and 54 (bound by stores of 4 bytes to lines of their own; loading further ahead changes nothing).

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
constexpr uint32_t kSmall = 16384, kSmallThreads = 1024, kSmallWaves = kSmallThreads / 64;
constexpr uint32_t kSmallBits = 9, kSmallDigits = 1u << kSmallBits;

// what a sort leaves behind
struct Sorted {
    int32_t* row;
    float* weight;                    // or null
    uint32_t* row_at;                 // of elements in their own order: one block's, where rows are ragged
    uint32_t *keys, *begin, *end;     // of the runs of equal keys, or null:
    uint32_t* start;                  // where every key's elements start, [n_keys + 1]
};
// A matrix to be cleared.  Measured over 512 MiB: pieces of 16 KiB a block of 256 threads 89 us, of 256 KiB a block of 1024 threads
// 88 us, all blocks side by side through the whole matrix 112 us, the runtime's own fill 83 us.
struct Fill {
    char* data;
    uint64_t n_rows, row_bytes, ld_bytes;
};
__device__ __forceinline__ void fill_rows(const Fill& f, uint64_t block, uint64_t blocks, uint32_t threads) {
    const auto clear = [](char* to, uint64_t bytes) {   // 16 of them, or what is left
        if (bytes >= 16) {
            *reinterpret_cast<Bytes16*>(to) = Bytes16{0, 0, 0, 0};
        } else {
            for (uint64_t k = 0; k < bytes; k += 2) *reinterpret_cast<uint16_t*>(to + k) = 0;
        }
    };
    if (f.row_bytes == f.ld_bytes) {   // one run of bytes, a piece a block
        const uint64_t n = f.n_rows * f.row_bytes, each = ((n + blocks - 1) / blocks + 15) / 16 * 16, first = block * each;
        const uint64_t end = first + each < n ? first + each : n;
        for (uint64_t at = first + threadIdx.x * 16; at < end; at += threads * 16) clear(f.data + at, end - at);
        return;
    }
    for (uint64_t r = block; r < f.n_rows; r += blocks)
        for (uint64_t at = threadIdx.x * 16; at < f.row_bytes; at += threads * 16) clear(f.data + r * f.ld_bytes + at, f.row_bytes - at);
}
__global__ __launch_bounds__(256) void k_fill(Fill f) { fill_rows(f, blockIdx.x, gridDim.x, 256); }

// Block 0 sorts up to TURNS * 1024 elements; the others clear the result meanwhile, where rows that no id names have to
// become zero.
template <uint32_t TURNS>
__global__ __launch_bounds__(kSmallThreads) void k_sort_small(SortArgs a, Sorted out, Fill fill) {
    if (blockIdx.x > 0) {
        fill_rows(fill, blockIdx.x - 1, gridDim.x - 1, kSmallThreads);
        return;
    }
    constexpr uint32_t kRoom = TURNS * kSmallThreads > kSmallDigits ? TURNS * kSmallThreads : kSmallDigits;
    __shared__ uint32_t key_at[kRoom];
    __shared__ uint16_t elem_at[TURNS * kSmallThreads];
    __shared__ uint32_t counter[kSmallWaves][kSmallDigits];
    __shared__ uint32_t digit_waves[kSmallDigits / 64], first_head[kSmallWaves], last_head[kSmallWaves];
    const uint32_t n = (uint32_t)a.n, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t turns = (n + kSmallThreads - 1) / kSmallThreads;   // a wave owns turns * 64 neighbouring elements
    uint32_t key[TURNS], elem[TURNS], place[TURNS];
#pragma unroll
    for (uint32_t t = 0; t < TURNS; ++t) {
        elem[t] = (wave * turns + t) * 64 + lane;
        key[t] = t < turns && elem[t] < n ? key_of(a, elem[t]) : 0u;
    }
    if (a.off) {
        // The rows, while neighbouring lanes still search for neighbouring elements, and in all turns at once (3450 elements of 1381
        // rows: 23.5 us, and 26.4 where sorted elements look for theirs)
        uint32_t row[TURNS] = {};
        for (uint64_t left = a.n_rows; left > 1;) {   // row[t]: the last of so many that starts at or before the element
            const uint32_t half = (uint32_t)(left >> 1);
#pragma unroll
            for (uint32_t t = 0; t < TURNS; ++t)
                if (t < turns) row[t] = a.off[row[t] + half] <= elem[t] ? row[t] + half : row[t];
            left -= half;
        }
#pragma unroll
        for (uint32_t t = 0; t < TURNS; ++t)
            if (t < turns && elem[t] < n) out.row_at[elem[t]] = row[t];
    }
    for (uint32_t shift = 0; shift < a.key_bits; shift += kSmallBits) {
        for (uint32_t k = threadIdx.x; k < kSmallWaves * kSmallDigits; k += kSmallThreads) counter[k >> kSmallBits][k & (kSmallDigits - 1)] = 0;
        __syncthreads();
#pragma unroll
        for (uint32_t t = 0; t < TURNS; ++t) {
            if (t >= turns) continue;
            // (positions, not elements, say which lanes are live: after the first pass the last ones are the largest keys)
            const bool live = (wave * turns + t) * 64 + lane < n;
            place[t] = rank_in_wave<kSmallBits>(counter[wave], (key[t] >> shift) & (kSmallDigits - 1), live);
        }
        __syncthreads();
        if (threadIdx.x < kSmallDigits) {   // a digit a thread: sums over the waves, then over the digits
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
        if (threadIdx.x < kSmallDigits) {
            uint32_t before = key_at[threadIdx.x];
            for (uint32_t w = 0; w < wave; ++w) before += digit_waves[w];
            for (uint32_t w = 0; w < kSmallWaves; ++w) counter[w][threadIdx.x] += before;
        }
        __syncthreads();
#pragma unroll
        for (uint32_t t = 0; t < TURNS; ++t) {
            if (t >= turns) continue;
            if ((wave * turns + t) * 64 + lane < n) {
                const uint32_t to = counter[wave][(key[t] >> shift) & (kSmallDigits - 1)] + place[t];
                key_at[to] = key[t];
                elem_at[to] = (uint16_t)elem[t];
            }
        }
        __syncthreads();
#pragma unroll
        for (uint32_t t = 0; t < TURNS; ++t) {
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
    for (uint32_t t = 0; t < TURNS; ++t) {
        if (t >= turns) continue;
        const uint32_t p = (wave * turns + t) * 64 + lane;
        if (p < n) {
            out.row[p] = (int32_t)(a.off ? out.row_at[elem[t]] : elem[t] / a.row_len);
            if (out.weight) out.weight[p] = a.weight[elem[t]];
            if (out.keys) out.keys[p] = key[t];
            key_at[p] = key[t];
        }
    }
    __syncthreads();
    if (out.start) {
        for (uint32_t v = threadIdx.x; v <= a.n_keys; v += kSmallThreads) {
            uint32_t lo = 0, hi = n;
            while (lo < hi) {
                const uint32_t mid = (lo + hi) >> 1;
                if (key_at[mid] < v) lo = mid + 1;
                else hi = mid;
            }
            out.start[v] = lo;
        }
        return;
    }
    // A run begins at the nearest head -- an element whose key differs from the one before -- at or before, and ends at the next
    // head after: found in the wave's ballots, and in the waves' first and last heads.
    unsigned long long heads[TURNS];
    uint32_t first = n, last = 0;
#pragma unroll
    for (uint32_t t = 0; t < TURNS; ++t) {
        heads[t] = 0;
        if (t >= turns) continue;
        const uint32_t p0 = (wave * turns + t) * 64, p = p0 + lane;
        heads[t] = __builtin_amdgcn_ballot_w64(p < n && (p == 0 || key_at[p - 1] != key[t]));
        if (heads[t]) {
            if (first == n) first = p0 + (uint32_t)__builtin_ctzll(heads[t]);
            last = p0 + 63 - (uint32_t)__builtin_clzll(heads[t]);
        }
    }
    if (lane == 0) {
        first_head[wave] = first;
        last_head[wave] = last;   // (0 is a head)
    }
    __syncthreads();
    uint32_t before = 0, after = n;
    for (uint32_t w = 0; w < kSmallWaves; ++w) {
        if (w < wave) before = last_head[w] > before ? last_head[w] : before;
        if (w > wave) after = first_head[w] < after ? first_head[w] : after;
    }
#pragma unroll
    for (uint32_t t = 0; t < TURNS; ++t) {
        if (t >= turns) continue;
        const uint32_t p0 = (wave * turns + t) * 64, p = p0 + lane;
        const unsigned long long upto = heads[t] & (~0ull >> (63 - lane));
        if (p < n) out.begin[p] = upto ? p0 + 63 - (uint32_t)__builtin_clzll(upto) : before;
        if (heads[t]) before = p0 + 63 - (uint32_t)__builtin_clzll(heads[t]);
    }
#pragma unroll
    for (uint32_t i = 0; i < TURNS; ++i) {
        const uint32_t t = TURNS - 1 - i;
        if (t >= turns) continue;
        const uint32_t p0 = (wave * turns + t) * 64, p = p0 + lane;
        const unsigned long long later = lane == 63 ? 0ull : heads[t] & (~0ull << (lane + 1));
        if (p < n) out.end[p] = later ? p0 + (uint32_t)__builtin_ctzll(later) : after;
        if (heads[t]) after = p0 + (uint32_t)__builtin_ctzll(heads[t]);
    }
}

constexpr uint32_t kTileWaves = 4, kMostDigits = 4096;   // of a tile of the sort of many elements

struct PassArgs {
    const uint32_t* keys;    // null in the first pass: the ids themselves
    const uint32_t* elems;
    uint32_t* counts;        // [tile][digit]
    uint32_t* totals;        // [digit]
    uint32_t shift, bits, turns, n_tiles;   // turns: of 64 elements a wave
    uint32_t last, only;     // the only pass sends nothing that does not contribute (a key of n_keys needs no digit), and hands on its keys alone
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
    for (uint64_t i = threadIdx.x; i < tile && t0 + i < a.n; i += 256) {
        const uint32_t key = pass_key(a, s, t0 + i);
        if (!s.only || key < a.n_keys) atomicAdd(&h[(key >> s.shift) & (digits - 1)], 1u);   // (a count does not depend on their order)
    }
    __syncthreads();
    for (uint32_t d = threadIdx.x; d < digits; d += 256) s.counts[(uint64_t)blockIdx.x * digits + d] = h[d];
}

// counts[tile][digit] become what the tiles before hold of the digit; totals[digit] what all do.  A block takes 64 digits, its
// eight waves sixteen tiles each at a time, all read at once.
constexpr uint32_t kSumWaves = 8, kSumTiles = 16;
__global__ __launch_bounds__(64 * kSumWaves) void k_sum_tiles(PassArgs s) {
    __shared__ uint32_t sums[kSumWaves][64];
    const uint32_t digits = 1u << s.bits, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, d = blockIdx.x * 64 + lane;   // (digits: a multiple of 64)
    uint32_t carry = 0;
    for (uint32_t t0 = 0; t0 < s.n_tiles; t0 += kSumWaves * kSumTiles) {
        const uint32_t first = t0 + wave * kSumTiles;
        uint32_t c[kSumTiles], sum = 0;
#pragma unroll
        for (uint32_t k = 0; k < kSumTiles; ++k) c[k] = first + k < s.n_tiles ? s.counts[(uint64_t)(first + k) * digits + d] : 0u;
#pragma unroll
        for (uint32_t k = 0; k < kSumTiles; ++k) sum += c[k];
        sums[wave][lane] = sum;
        __syncthreads();
        uint32_t before = carry;
        for (uint32_t w = 0; w < kSumWaves; ++w) {
            before += w < wave ? sums[w][lane] : 0u;
            carry += sums[w][lane];
        }
        __syncthreads();
#pragma unroll
        for (uint32_t k = 0; k < kSumTiles; ++k) {
            if (first + k < s.n_tiles) s.counts[(uint64_t)(first + k) * digits + d] = before;
            before += c[k];
        }
    }
    if (wave == 0) s.totals[d] = carry;
}

template <int BITS>
__global__ __launch_bounds__(256) void k_scatter(SortArgs a, PassArgs s) {
    constexpr uint32_t kDigits = 1u << BITS, kEach = (kDigits + 255) / 256;   // digits of a thread
    __shared__ uint32_t next[kTileWaves][kDigits];
    __shared__ uint32_t sums[kEach * 4 + 1];   // the last one: of all digits
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
        if (p < a.n) {
            const uint32_t key = pass_key(a, s, p);
            if (!s.only || key < a.n_keys) atomicAdd(&next[wave][(key >> s.shift) & (kDigits - 1)], 1u);
        }
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
        if (lane == 63) sums[kEach * 4] = sum;
    }
    __syncthreads();
    // The places behind what the only pass sends hold the key of what contributes nothing: a list that is searched for its runs has
    // to be sorted to its end.  (All tiles write some of them; no row or weight is read there.)
    if (s.only && s.keys_out)
        for (uint64_t p = sums[kEach * 4] + (uint64_t)blockIdx.x * 256 + threadIdx.x; p < a.n; p += (uint64_t)gridDim.x * 256) s.keys_out[p] = (uint32_t)a.n_keys;
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) {
        const uint32_t d = i * 256 + threadIdx.x;
        if (d >= kDigits) continue;
        first[i] += sums[i * 4 + wave];
        if (s.start && blockIdx.x == 0) {
            if (d < a.n_keys) s.start[d] = first[i];
            if (d + 1 == a.n_keys) s.start[a.n_keys] = first[i] + total[i];
        }
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
        const uint32_t key = p < a.n ? pass_key(a, s, p) : 0u;
        const bool live = p < a.n && (!s.only || key < a.n_keys);
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

// where the run of equal keys around every sorted position begins and ends
__global__ __launch_bounds__(256) void k_runs(const uint32_t* __restrict__ keys, uint64_t first, uint64_t n, uint32_t* __restrict__ begin,
                                              uint32_t* __restrict__ end) {
    const uint64_t p = first + (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (p >= n) return;
    const uint32_t key = keys[p];
    uint64_t lo = 0, hi = p;   // first position whose key is `key`
    while (lo < hi) {
        const uint64_t mid = (lo + hi) >> 1;
        if (keys[mid] < key) lo = mid + 1;
        else hi = mid;
    }
    begin[p] = (uint32_t)lo;
    lo = p + 1;
    hi = n;
    while (lo < hi) {
        const uint64_t mid = (lo + hi) >> 1;
        if (keys[mid] <= key) lo = mid + 1;
        else hi = mid;
    }
    end[p] = (uint32_t)lo;
}

// ---- the gradient to the weights ------------------------------------------------------------------------------------------
// A wave takes 8 or 16 elements, a lane finding the row and the table row of each, and works through them B at a time: every lane
// loads 16 bytes of the B table rows and of their gradients' row, column after column, and the B sums over the lanes are
// formed together: in three steps eight values a lane become one value an eighth of the lanes, half of the values changing
// sides each time.  Bound: instruction issue (16 of a table row's 16 bytes' conversions and products) and L2.  Measured: 8192 rows of
// 40 elements of 512 bf16 columns (336 MB of table rows read) in 22.5 us = 15 TB/s.
// (On the matrix cores, as the diagonal of sixteen rows times sixteen rows, the same takes 48 us where this takes 23 (8192 x 40
// dot products of 512 bf16): what a lane has to load there are 16 bytes of a row of its own, and L1 looks up a line for each.)

// ALIGNED: rows hold a multiple of B elements each, so that B neighbours always share theirs
template <bool ALIGNED, typename T, typename G>
__global__ __launch_bounds__(256) void k_weight_grad(SortArgs a, uint64_t first, uint32_t dots, const G* __restrict__ grad, uint64_t grad_ld, const T* __restrict__ table,
                                                     uint64_t table_ld, uint32_t dim, float scale, float* __restrict__ out) {
    constexpr int V = 16 / (sizeof(T) > sizeof(G) ? sizeof(T) : sizeof(G)), B = 8;
    const uint64_t e0 = first + ((uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * dots;
    const uint32_t lane = threadIdx.x & 63;
    if (e0 >= a.n) return;
    uint32_t id = (uint32_t)a.n_keys, row = 0;
    if (lane < dots && e0 + lane < a.n) id = key_of(a, e0 + lane);
    if (a.off) {
        // the row of the first one, and how many of the next 64 rows start at or before the others
        const uint64_t row0 = segment_at(a.off, a.n_rows, e0), next = row0 + 1 + lane;
        const uint64_t begins = next <= a.n_rows ? a.off[next] : ~0ull;
        uint32_t passed = 0;
        for (uint32_t u = 0; u < dots; ++u) {
            const uint32_t k = (uint32_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64(begins <= e0 + u));
            if (lane == u) passed = k;
        }
        row = (uint32_t)row0 + passed;
        if (passed == 64) row = row_of(a.off, a.n_rows, a.row_len, e0 + lane);   // (many empty rows)
        row = row < a.n_rows ? row : 0;   // (behind the last row: an element that contributes nothing)
    } else {
        row = (uint32_t)(e0 + lane) / a.row_len;
        row = row < a.n_rows ? row : 0;
    }
    const unsigned long long live = __builtin_amdgcn_ballot_w64(id < a.n_keys);
    if (id >= a.n_keys) id = 0;   // (where any element is live, the matrices have rows)
    float mine = 0.0f;            // of the lane's own element
    for (uint32_t u = 0; u < dots; u += B) {
        if (((live >> u) & 0xFFu) == 0) continue;
        const T* t[B];
        uint32_t r[B];
        bool one_row = true;
#pragma unroll
        for (int j = 0; j < B; ++j) {
            t[j] = table + (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)id, (int)u + j) * table_ld;
            r[j] = (uint32_t)__builtin_amdgcn_readlane((int)row, (int)u + j);
            one_row = one_row && (ALIGNED || r[j] == r[0]);
        }
        float sum[B] = {};
        const G* g = grad + (uint64_t)r[0] * grad_ld;
#pragma unroll 1
        for (uint32_t c = lane * V; c < dim; c += 64 * V) {
            if (c + V <= dim) {
                T x[B][V];
#pragma unroll
                for (int j = 0; j < B; ++j) load_n<V>(t[j] + c, x[j]);
                if (ALIGNED || one_row) {
                    G y[V];
                    load_n<V>(g + c, y);
#pragma unroll
                    for (int j = 0; j < B; ++j)
#pragma unroll
                        for (int k = 0; k < V; ++k) sum[j] = fmaf(to_f32(x[j][k]), to_f32(y[k]), sum[j]);
                } else {
                    G y[B][V];
#pragma unroll
                    for (int j = 0; j < B; ++j) load_n<V>(grad + (uint64_t)r[j] * grad_ld + c, y[j]);
#pragma unroll
                    for (int j = 0; j < B; ++j)
#pragma unroll
                        for (int k = 0; k < V; ++k) sum[j] = fmaf(to_f32(x[j][k]), to_f32(y[j][k]), sum[j]);
                }
            } else {
                for (uint32_t k = c; k < dim; ++k)
#pragma unroll
                    for (int j = 0; j < B; ++j)
                        sum[j] = fmaf(to_f32(t[j][k]), to_f32(ALIGNED ? g[k] : grad[(uint64_t)r[j] * grad_ld + k]), sum[j]);
            }
        }
        // lane bits 3, 2 and 1 choose which half of the values a lane keeps; the other half comes from the lane across
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float keep = lane & 8 ? sum[2 * j + 1] : sum[2 * j], give = lane & 8 ? sum[2 * j] : sum[2 * j + 1];
            sum[j] = keep + dpp<0x140, 0xF>(give, give);   // 15 - lane in a row of 16
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float keep = lane & 4 ? sum[2 * j + 1] : sum[2 * j], give = lane & 4 ? sum[2 * j] : sum[2 * j + 1];
            sum[j] = keep + dpp<0x141, 0xF>(give, give);   // 7 - lane
        }
        {
            const float keep = lane & 2 ? sum[1] : sum[0], give = lane & 2 ? sum[0] : sum[1];
            sum[0] = keep + dpp<0x1B, 0xF>(give, give);    // 3 - lane
        }
        sum[0] += dpp<0xB1, 0xF>(sum[0], sum[0]);          // 1 - lane
        sum[0] += __shfl_xor(sum[0], 16, 64);
        sum[0] += __shfl_xor(sum[0], 32, 64);
        // bit 0 of an element lies in lane bit 3, bit 1 in bit 2, bit 2 in bit 1
        const float dot = __shfl(sum[0], (int)((lane & 1) * 8 + (lane & 2) * 2 + (lane & 4) / 2), 64);
        if ((lane & ~7u) == u) mine = scale * dot;
    }
    if (lane < dots && e0 + lane < a.n) out[e0 + lane] = (live >> lane) & 1 ? mine : 0.0f;
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
    Passes(uint64_t n, uint64_t n_keys) {
        const uint32_t key_bits = n_keys && n_keys <= kMostDigits ? bits_of(n_keys - 1) : bits_of(n_keys);   // (one pass needs no key of n_keys)
        turns = 2;
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

// How the table's gradient is put together, and what it keeps in the caller's scratch.  Fewer than three elements an id on average
// (tokens): the runs of the sorted list are summed, and the result is cleared first -- by the blocks that the sort does not
// need, where one block sorts.  More (codes): the ids are the segments, and those without elements write their zeros.
struct Plan {
    bool runs, small;
    uint32_t chunk;
    Sorted sorted;
    uint32_t *keys[2], *elems[2], *counts, *totals;
    float* partials;
    size_t bytes;
    Plan(void* base, uint64_t n, uint64_t n_keys, bool weighted, bool ragged, uint32_t dim) {
        size_t at = 0;
        const auto take = [&](size_t count) {
            char* p = static_cast<char*>(base) + (base ? at : 0);
            at += up(count * 4);
            return reinterpret_cast<uint32_t*>(p);
        };
        const Passes p(n, n_keys);
        runs = n < 3 * n_keys;
        // One block, or three launches a pass: 4096 elements of 2048 ids 19 us against 24, 8192 29 against 18; 8192 of 5000
        // ids (two passes) 31 either way, 16384 44 against 31.  While a large result is cleared one block's time is hidden:
        // 16384 with 537 MB to clear 135 us against 160, with 134 MB 77 against 75.
        small = n <= 4096ull * p.count || (runs && n <= kSmall && n_keys * dim >= 1ull << 25);
        chunk = runs ? run_chunk(n) : segment_chunk(n_keys, n, dim, true);
        sorted.row = reinterpret_cast<int32_t*>(take(n));
        sorted.weight = weighted ? reinterpret_cast<float*>(take(n)) : nullptr;
        sorted.row_at = take(small && ragged ? n : 0);
        // what the passes hand on; the last one's keys where runs or starts are looked for in them
        const bool keep = runs || (!small && p.count > 1);
        for (uint32_t k = 0; k < 2; ++k) {
            const bool last = (p.count - 1) % 2 == k;
            keys[k] = take(small ? (k == 0 && keep ? n : 0) : p.count > 1 + k || (last && keep) ? n : 0);
            elems[k] = take(!small && p.count > 1 + k ? n : 0);
        }
        sorted.keys = keep ? keys[small ? 0 : (p.count - 1) % 2] : nullptr;
        sorted.begin = runs ? take(n) : nullptr;
        sorted.end = runs ? take(n) : nullptr;
        sorted.start = runs ? nullptr : take(n_keys + 1);
        counts = take(small ? 0 : (size_t)p.n_tiles << p.bits);
        totals = take(small ? 0 : (size_t)1 << p.bits);
        partials = reinterpret_cast<float*>(take(0));
        bytes = at + partial_bytes(chunk, n, dim);
    }
};

int sort_by_id(const SortArgs& a, const Plan& s, const Fill& fill, hipStream_t stream) {
    const uint64_t to_fill = s.runs ? fill.n_rows * fill.row_bytes : 0;
    if (s.small) {
        const uint32_t blocks = (uint32_t)std::min<uint64_t>((to_fill + 262143) / 262144, 1u << 20);
        const auto sort = a.n <= kSmallThreads ? &k_sort_small<1> : a.n <= 4 * kSmallThreads ? &k_sort_small<4> : &k_sort_small<16>;
        hipLaunchKernelGGL(sort, dim3(1 + blocks), dim3(kSmallThreads), 0, stream, a, s.sorted, fill);
        SDRB_HIP(hipGetLastError());
        return SDRB_OK;
    }
    if (to_fill) {
        hipLaunchKernelGGL(k_fill, dim3((uint32_t)std::min<uint64_t>((to_fill + 16383) / 16384, 1u << 20)), dim3(256), 0, stream, fill);
        SDRB_HIP(hipGetLastError());
    }
    const Passes passes(a.n, a.n_keys);
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
        p.only = passes.count == 1;
        p.keys_out = p.last ? s.sorted.keys : s.keys[k & 1];
        p.elems_out = s.elems[k & 1];
        p.row_out = s.sorted.row;
        p.weight_out = s.sorted.weight;
        p.start = passes.count == 1 ? s.sorted.start : nullptr;
        hipLaunchKernelGGL(k_count, dim3(passes.n_tiles), dim3(256), 0, stream, a, p);
        SDRB_HIP(hipGetLastError());
        hipLaunchKernelGGL(k_sum_tiles, dim3((1u << passes.bits) / 64), dim3(64 * kSumWaves), 0, stream, p);
        SDRB_HIP(hipGetLastError());
        const auto scatter = passes.bits == 12   ? &k_scatter<12>
                             : passes.bits == 11 ? &k_scatter<11>
                             : passes.bits == 10 ? &k_scatter<10>
                             : passes.bits == 9  ? &k_scatter<9>
                                                 : &k_scatter<8>;
        hipLaunchKernelGGL(scatter, dim3(passes.n_tiles), dim3(256), 0, stream, a, p);
        SDRB_HIP(hipGetLastError());
    }
    if (s.runs) {
        return in_launches((a.n + 255) / 256, 256, [&](uint64_t first, uint32_t blocks) {
            hipLaunchKernelGGL(k_runs, dim3(blocks), dim3(256), 0, stream, s.sorted.keys, first * 256, a.n, s.sorted.begin, s.sorted.end);
            SDRB_HIP(hipGetLastError());
            return SDRB_OK;
        });
    }
    if (passes.count > 1) {
        hipLaunchKernelGGL(k_starts, dim3((uint32_t)(a.n_keys / 256 + 1)), dim3(256), 0, stream, s.sorted.keys, a.n, a.n_keys, s.sorted.start);
        SDRB_HIP(hipGetLastError());
    }
    return SDRB_OK;
}

}  // namespace

size_t table_grad_scratch_bytes(const sdrb_rows& rows, uint64_t n_table_rows, uint32_t dim) {
    return Plan(nullptr, rows.n_elems, n_table_rows, rows.weights != nullptr, rows.row_offsets != nullptr, dim).bytes;
}

int launch_table_grad(const sdrb_rows& rows, const sdrb_dense& grad, float scale, bool accumulate, const sdrb_dense& out, void* scratch,
                      hipStream_t stream) {
    const uint32_t dim = (uint32_t)out.n_cols;
    const Plan plan(scratch, rows.n_elems, out.n_rows, rows.weights != nullptr, rows.row_offsets != nullptr, dim);
    const SortArgs a = sort_args(rows, out.n_rows);
    const size_t size = type_size(out.type);
    const Fill fill{static_cast<char*>(out.data), accumulate ? 0 : out.n_rows, dim * size, out.ld * size};
    if (const int rc = sort_by_id(a, plan, fill, stream)) return rc;
    if (plan.runs && rows.n_elems == 0) return SDRB_OK;
    GatherSum g{};
    g.n_segments = plan.runs ? rows.n_elems : out.n_rows;
    g.n_elems = rows.n_elems;
    g.start = plan.sorted.start;
    if (plan.runs) {
        g.keys = plan.sorted.keys;
        g.begin = plan.sorted.begin;
        g.end = plan.sorted.end;
    }
    g.out_rows = out.n_rows;
    g.index = plan.sorted.row;
    g.index_bits = 32;
    g.weight = plan.sorted.weight;
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
    g.chunk = plan.chunk;
    g.partials = plan.partials;
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
            const auto kernel = !a.off && a.row_len % 8 == 0 ? &k_weight_grad<true, T, G> : &k_weight_grad<false, T, G>;
            // of a wave: more of them wait less for the rows and ids of the first, fewer make more waves.  8 against 16 and 32: 1408 of
            // 1728 columns 6.3, 10.1 and 17.8 us, 65536 of 512 7.1, 6.8 and 8.1, 262144 20.3, 18.3 and 19.3
            const uint32_t dots = a.n < 65536 ? 8 : 16;
            return in_launches((a.n + 4 * dots - 1) / (4 * dots), 256, [&](uint64_t first, uint32_t blocks) {
                hipLaunchKernelGGL(kernel, dim3(blocks), dim3(256), 0, stream, a, first * 4 * dots, dots, static_cast<const G*>(grad.data), grad.ld,
                                   static_cast<const T*>(table.data), table.ld, (uint32_t)table.n_cols, scale, out);
                SDRB_HIP(hipGetLastError());
                return SDRB_OK;
            });
        });
    });
}

}  // namespace sdrb
