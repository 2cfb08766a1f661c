// Gradients of a lookup out[r, :] = scale * sum over row r's elements e of w[e] * table[id[e], :].
//
// To the table: d table[v, :] = scale * sum over the elements e with id[e] = v of w[e] * d out[row(e), :].  The elements are
// sorted by id -- a stable radix sort, so that the elements of one id keep their order -- and the sums run over the
// sorted list like a lookup whose rows are the ids (lookup.hip): no atomic addition, the same bits every time, and the
// work of an id that many rows hold is shared out.
// To the weights: d w[e] = scale * <d out[row(e), :], table[id[e], :]>, a dot product an element.
#include "dense_rows.h"

namespace sdrb {

namespace {

constexpr uint32_t kTile = 2048, kDigitBits = 8, kDigits = 1u << kDigitBits, kWaves = 4, kPerWave = kTile / kWaves;

// the row of element e
__device__ __forceinline__ uint32_t row_of(const uint32_t* __restrict__ off, uint64_t n_rows, uint32_t row_len, uint64_t e) {
    if (!off) return (uint32_t)(e / row_len);
    uint64_t lo = 0, hi = n_rows;   // last row that starts at or before e
    while (hi - lo > 1) {
        const uint64_t mid = (lo + hi) >> 1;
        if (off[mid] <= e) lo = mid;
        else hi = mid;
    }
    return (uint32_t)lo;
}

// Elements as sort keys: the id, or n_table_rows for an element that contributes nothing (an id outside the table, or an
// element behind the last row).
template <typename Id>
__global__ __launch_bounds__(256) void k_keys(const Id* __restrict__ ids, uint64_t n, uint64_t n_table_rows,
                                              const uint32_t* __restrict__ off, uint64_t n_rows, uint32_t* __restrict__ keys,
                                              uint32_t* __restrict__ elems) {
    const uint64_t e = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (e >= n) return;
    const Id id = ids[e];
    const bool in = id >= 0 && (uint64_t)id < n_table_rows && (!off || (e >= off[0] && e < off[n_rows]));
    keys[e] = in ? (uint32_t)id : (uint32_t)n_table_rows;
    elems[e] = (uint32_t)e;
}

// counts[digit * n_tiles + tile]: keys of the tile whose digit is `digit`
__global__ __launch_bounds__(256) void k_count(const uint32_t* __restrict__ keys, uint64_t n, uint32_t shift, uint32_t n_tiles,
                                               uint32_t* __restrict__ counts) {
    __shared__ uint32_t h[kDigits];
    h[threadIdx.x] = 0;
    __syncthreads();
    const uint64_t t0 = (uint64_t)blockIdx.x * kTile;
    for (uint32_t i = threadIdx.x; i < kTile && t0 + i < n; i += 256) atomicAdd(&h[(keys[t0 + i] >> shift) & (kDigits - 1)], 1u);
    __syncthreads();
    counts[(uint64_t)threadIdx.x * n_tiles + blockIdx.x] = h[threadIdx.x];
}

// in-place exclusive prefix sum by one block
__global__ __launch_bounds__(1024) void k_scan(uint32_t* __restrict__ data, uint64_t n) {
    __shared__ uint32_t waves[16];
    uint32_t carry = 0;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (uint64_t base = 0; base < n; base += 1024) {
        const uint64_t i = base + threadIdx.x;
        const uint32_t v = i < n ? data[i] : 0u;
        uint32_t sum = v;
#pragma unroll
        for (uint32_t s = 1; s < 64; s <<= 1) {
            const uint32_t below = (uint32_t)__shfl_up((int)sum, s, 64);
            if (lane >= s) sum += below;
        }
        if (lane == 63) waves[wave] = sum;
        __syncthreads();
        uint32_t before = 0, total = 0;
        for (uint32_t k = 0; k < 16; ++k) {
            before += k < wave ? waves[k] : 0u;
            total += waves[k];
        }
        if (i < n) data[i] = carry + before + sum - v;
        carry += total;
        __syncthreads();
    }
}

// Sends the tile's pairs to their digits' places, in order.  Within a wave the 64 elements of a turn find the others of
// their digit by a ballot a key bit; a wave's first place of a digit is the tile's plus what the waves before it hold.
__global__ __launch_bounds__(256) void k_scatter(const uint32_t* __restrict__ keys, const uint32_t* __restrict__ elems, uint64_t n,
                                                 uint32_t shift, uint32_t n_tiles, const uint32_t* __restrict__ starts,
                                                 uint32_t* __restrict__ keys_out, uint32_t* __restrict__ elems_out) {
    __shared__ uint32_t next[kWaves][kDigits];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (uint32_t k = 0; k < kWaves; ++k) next[k][threadIdx.x] = 0;
    __syncthreads();
    const uint64_t w0 = (uint64_t)blockIdx.x * kTile + wave * kPerWave;
    for (uint32_t i = lane; i < kPerWave && w0 + i < n; i += 64) atomicAdd(&next[wave][(keys[w0 + i] >> shift) & (kDigits - 1)], 1u);
    __syncthreads();
    {
        uint32_t at = starts[(uint64_t)threadIdx.x * n_tiles + blockIdx.x];
        for (uint32_t k = 0; k < kWaves; ++k) {
            const uint32_t here = next[k][threadIdx.x];
            next[k][threadIdx.x] = at;
            at += here;
        }
    }
    __syncthreads();
    for (uint32_t i0 = 0; i0 < kPerWave; i0 += 64) {   // the same number of turns for every wave
        const uint64_t p = w0 + i0 + lane;
        const bool live = p < n;
        const uint32_t key = live ? keys[p] : 0u, elem = live ? elems[p] : 0u;
        const uint32_t digit = (key >> shift) & (kDigits - 1);
        unsigned long long same = __builtin_amdgcn_ballot_w64(live);
#pragma unroll
        for (uint32_t b = 0; b < kDigitBits; ++b) {
            const unsigned long long set = __builtin_amdgcn_ballot_w64((digit >> b) & 1u);
            same &= ((digit >> b) & 1u) ? set : ~set;
        }
        const uint32_t rank = (uint32_t)__builtin_popcountll(same & ((1ull << lane) - 1ull));
        const uint32_t place = live ? next[wave][digit] + rank : 0u;
        __syncthreads();   // all have read their digit's place
        if (live && rank == 0) next[wave][digit] += (uint32_t)__builtin_popcountll(same);
        __syncthreads();
        if (live) {
            keys_out[place] = key;
            elems_out[place] = elem;
        }
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

// the sorted elements' rows and weights
__global__ __launch_bounds__(256) void k_rows(const uint32_t* __restrict__ elems, uint64_t n, const uint32_t* __restrict__ off,
                                              uint64_t n_rows, uint32_t row_len, const float* __restrict__ weight,
                                              int32_t* __restrict__ row, float* __restrict__ row_weight) {
    const uint64_t p = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (p >= n) return;
    const uint32_t e = elems[p];
    row[p] = (int32_t)row_of(off, n_rows, row_len, e);
    if (weight) row_weight[p] = weight[e];
}

// one wave per element: the dot product of its row's gradient and its table row
template <typename T, typename G, typename Id>
__global__ __launch_bounds__(256) void k_weight_grad(const Id* __restrict__ ids, uint64_t n, const uint32_t* __restrict__ off,
                                                     uint64_t n_rows, uint32_t row_len, const G* __restrict__ grad, uint64_t grad_ld,
                                                     const T* __restrict__ table, uint64_t table_rows, uint64_t table_ld, uint32_t dim,
                                                     float scale, float* __restrict__ out) {
    const uint64_t e = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const uint32_t lane = threadIdx.x & 63;
    if (e >= n) return;
    const Id id = ids[e];
    float sum = 0.0f;
    const bool in = id >= 0 && (uint64_t)id < table_rows && (!off || (e >= off[0] && e < off[n_rows]));
    if (in) {
        const G* g = grad + (uint64_t)row_of(off, n_rows, row_len, e) * grad_ld;
        const T* t = table + (uint64_t)id * table_ld;
        for (uint32_t c = lane; c < dim; c += 64) sum = fmaf(to_f32(g[c]), to_f32(t[c]), sum);
    }
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1) sum += __shfl_xor(sum, s, 64);
    if (lane == 0) out[e] = in ? scale * sum : 0.0f;
}

size_t up(size_t bytes) { return (bytes + 255) / 256 * 256; }

}  // namespace

size_t table_grad_scratch_bytes(uint64_t n_elems, uint64_t n_table_rows, uint32_t dim) {
    const size_t list = up(n_elems * sizeof(uint32_t));
    const size_t n_tiles = (n_elems + kTile - 1) / kTile;
    return 4 * list + up(n_tiles * kDigits * sizeof(uint32_t)) + up((n_table_rows + 1) * sizeof(uint32_t)) +
           gather_partial_bytes(n_table_rows, n_elems, true, dim);
}

int launch_table_grad(int device, const sdrb_rows& rows, const sdrb_dense& grad, float scale, bool accumulate, const sdrb_dense& out,
                      void* scratch, hipStream_t stream) {
    const uint64_t n = rows.n_elems, v = out.n_rows;
    const uint32_t dim = (uint32_t)out.n_cols, row_len = rows.row_offsets || !rows.n_rows ? 1u : (uint32_t)(n / rows.n_rows);
    const uint32_t n_tiles = (uint32_t)((n + kTile - 1) / kTile);
    char* ws = static_cast<char*>(scratch);
    const auto take = [&](size_t bytes) {
        char* p = ws;
        ws += up(bytes);
        return p;
    };
    uint32_t* keys[2];
    uint32_t* elems[2];
    for (int k = 0; k < 2; ++k) {
        keys[k] = reinterpret_cast<uint32_t*>(take(n * sizeof(uint32_t)));
        elems[k] = reinterpret_cast<uint32_t*>(take(n * sizeof(uint32_t)));
    }
    uint32_t* counts = reinterpret_cast<uint32_t*>(take((size_t)n_tiles * kDigits * sizeof(uint32_t)));
    uint32_t* start = reinterpret_cast<uint32_t*>(take((v + 1) * sizeof(uint32_t)));
    float* partials = gather_partial_bytes(v, n, true, dim) ? reinterpret_cast<float*>(ws) : nullptr;
    const dim3 per_elem((uint32_t)((n + 255) / 256));
    int now = 0;
    if (n) {
        if (rows.id_bits == 64)
            hipLaunchKernelGGL((k_keys<int64_t>), per_elem, dim3(256), 0, stream, static_cast<const int64_t*>(rows.ids), n, v,
                               rows.row_offsets, rows.n_rows, keys[0], elems[0]);
        else
            hipLaunchKernelGGL((k_keys<int32_t>), per_elem, dim3(256), 0, stream, static_cast<const int32_t*>(rows.ids), n, v,
                               rows.row_offsets, rows.n_rows, keys[0], elems[0]);
        SDRB_HIP(hipGetLastError());
        for (uint32_t shift = 0; shift < 32 && (v >> shift) != 0; shift += kDigitBits) {   // the largest key is v
            hipLaunchKernelGGL(k_count, dim3(n_tiles), dim3(256), 0, stream, keys[now], n, shift, n_tiles, counts);
            SDRB_HIP(hipGetLastError());
            hipLaunchKernelGGL(k_scan, dim3(1), dim3(1024), 0, stream, counts, (uint64_t)n_tiles * kDigits);
            SDRB_HIP(hipGetLastError());
            hipLaunchKernelGGL(k_scatter, dim3(n_tiles), dim3(256), 0, stream, keys[now], elems[now], n, shift, n_tiles, counts,
                               keys[now ^ 1], elems[now ^ 1]);
            SDRB_HIP(hipGetLastError());
            now ^= 1;
        }
    }
    hipLaunchKernelGGL(k_starts, dim3((uint32_t)(v / 256 + 1)), dim3(256), 0, stream, keys[now], n, v, start);
    SDRB_HIP(hipGetLastError());
    int32_t* row = reinterpret_cast<int32_t*>(keys[now ^ 1]);
    float* weight = rows.weights ? reinterpret_cast<float*>(elems[now ^ 1]) : nullptr;
    if (n) {
        hipLaunchKernelGGL(k_rows, per_elem, dim3(256), 0, stream, elems[now], n, rows.row_offsets, rows.n_rows, row_len, rows.weights,
                           row, weight);
        SDRB_HIP(hipGetLastError());
    }
    GatherSum g{};
    g.device = device;
    g.n_segments = v;
    g.n_elems = n;
    g.start = start;
    g.index = row;
    g.index_bits = 32;
    g.weight = weight;
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
    g.partials = partials;
    return launch_gather_sum(g, stream);
}

int launch_weight_grad(const sdrb_rows& rows, const sdrb_dense& grad, const sdrb_dense& table, float scale, float* out,
                       hipStream_t stream) {
    const uint64_t n = rows.n_elems;
    if (n == 0) return SDRB_OK;
    const uint32_t row_len = rows.row_offsets || !rows.n_rows ? 1u : (uint32_t)(n / rows.n_rows);
    return with_type(table.type, [&](auto t) {
        return with_type(grad.type, [&](auto g) {
            using T = decltype(t);
            using G = decltype(g);
            const auto go = [&](auto id) {
                using Id = decltype(id);
                hipLaunchKernelGGL((k_weight_grad<T, G, Id>), dim3((uint32_t)((n + 3) / 4)), dim3(256), 0, stream,
                                   static_cast<const Id*>(rows.ids), n, rows.row_offsets, rows.n_rows, row_len,
                                   static_cast<const G*>(grad.data), grad.ld, static_cast<const T*>(table.data), table.n_rows, table.ld,
                                   (uint32_t)table.n_cols, scale, out);
                SDRB_HIP(hipGetLastError());
                return SDRB_OK;
            };
            return rows.id_bits == 64 ? go(int64_t{}) : go(int32_t{});
        });
    });
}

}  // namespace sdrb
