// The k winners of every row of dense scores, with their weights, and the gradient of those weights to the scores.
//
// Shares: u = softmax of a row's live scores, or their sigmoids; a score of -inf or NaN is not live.  Keys: u + bias, or the
// scores where nothing is added to the shares (the same order).  A group's score is the sum of its one or two largest
// keys; the k largest keys inside the best groups win, ties go to the lowest group and id.
// Weights: scale * u, or, renormalised, scale * p with p = u / sum of the winners' u -- a softmax over the winners of
// l = s (softmax) or l = log sigmoid(s), which holds where every u underflows.
//
// A wave owns a row and holds its scores in registers, R a lane, read once; rows of more than 2048 ids are shared by eight
// waves.  Two steps choose the winners:
//  1. Candidates.  Of the lanes' largest keys a threshold is found that k of them reach (a compare and a population count a
//     step), so at least k keys reach it, and few more: about 62 of 2048 for k = 40.  Keys are binary32 here; where shares
//     enter them the threshold is lowered by what their arithmetic can be off, so that no winner is lost.
//  2. The candidates' ids go to LDS in ascending order, one a thread from there on; their keys are computed exactly, and the
//     k-th largest is found by bisection over the keys' order-preserving integers, which ends as soon as exactly k keys lie
//     at or above the middle.
// Shares that enter keys are computed in binary64 in the second step: whether an id wins hangs on the difference of two keys,
// which binary32 exponentials would decide by their own error.  Rows whose candidates are too many (many equal scores, a k
// near the number of lanes) or whose groups cannot be told apart in binary32 bisect over all their keys instead.
// Bound: instruction issue, not memory.
#include <type_traits>

#include "dense_rows.h"

namespace sdrb {

namespace {

// ---- a wave's reductions, by data-parallel moves: 6 steps without LDS ----
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp(int other, int v) {
    return __builtin_amdgcn_update_dpp(other, v, CTRL, ROWS, 0xF, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp(float other, float v) {
    return __builtin_bit_cast(float, dpp<CTRL, ROWS>(__builtin_bit_cast(int, other), __builtin_bit_cast(int, v)));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp(double other, double v) {
    const long long o = __builtin_bit_cast(long long, other), x = __builtin_bit_cast(long long, v);
    const uint32_t lo = (uint32_t)dpp<CTRL, ROWS>((int)o, (int)x), hi = (uint32_t)dpp<CTRL, ROWS>((int)(o >> 32), (int)(x >> 32));
    return __builtin_bit_cast(double, (long long)(((uint64_t)hi << 32) | lo));
}
__device__ __forceinline__ int last_lane(int v) { return __builtin_amdgcn_readlane(v, 63); }
__device__ __forceinline__ float last_lane(float v) { return __builtin_bit_cast(float, last_lane(__builtin_bit_cast(int, v))); }
__device__ __forceinline__ double last_lane(double v) {
    const long long x = __builtin_bit_cast(long long, v);
    const uint32_t lo = (uint32_t)last_lane((int)x), hi = (uint32_t)last_lane((int)(x >> 32));
    return __builtin_bit_cast(double, (long long)(((uint64_t)hi << 32) | lo));
}
// `none` leaves every value as it is under op; the result is uniform
template <typename T, typename F>
__device__ __forceinline__ T wave_reduce(T v, T none, F op) {
    v = op(v, dpp<0xB1, 0xF>(v, v));        // lanes 1 0 3 2
    v = op(v, dpp<0x4E, 0xF>(v, v));        // lanes 2 3 0 1
    v = op(v, dpp<0x141, 0xF>(v, v));       // the other half of 8
    v = op(v, dpp<0x140, 0xF>(v, v));       // the other half of 16
    v = op(v, dpp<0x142, 0xA>(none, v));    // lane 15 of the row of 16 below, into rows 1 and 3
    v = op(v, dpp<0x143, 0xC>(none, v));    // lane 31, into rows 2 and 3
    return last_lane(v);
}
template <typename T>
__device__ __forceinline__ T max_of(T a, T b) {
    return a > b ? a : b;
}

// ---- the waves of a row: WAVES == 1, or 8 that meet in LDS ----
template <int WAVES>
struct Meet {
    double* slot;   // [2][WAVES] where WAVES > 1
    uint32_t turn;

    template <typename T, typename F>
    __device__ __forceinline__ T all(T v, F op) {   // v: uniform in the wave
        if constexpr (WAVES == 1) {
            return v;
        } else {
            double* s = slot + (turn++ & 1) * WAVES;   // the turn before may still be read while this one is written
            if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = (double)v;
            __syncthreads();
            T r = (T)s[0];
#pragma unroll
            for (int k = 1; k < WAVES; ++k) r = op(r, (T)s[k]);
            return r;
        }
    }
    template <typename T>
    __device__ __forceinline__ T sum(T v) {
        return all(wave_reduce(v, T(0), [](T a, T b) { return a + b; }), [](T a, T b) { return a + b; });
    }
    template <typename T>
    __device__ __forceinline__ T max(T v) {
        return all(wave_reduce(v, (T)-INFINITY, max_of<T>), max_of<T>);
    }
    __device__ __forceinline__ uint32_t total(uint32_t uniform) {
        return all(uniform, [](uint32_t a, uint32_t b) { return a + b; });
    }
};

// ---- keys as integers of the same order ----
template <typename K>
struct Ordered;
template <>
struct Ordered<float> {
    using U = uint32_t;
    static constexpr U kSign = 0x80000000u;
};
template <>
struct Ordered<double> {
    using U = uint64_t;
    static constexpr U kSign = 0x8000000000000000ull;
};
template <typename K>
__device__ __forceinline__ typename Ordered<K>::U order_of(K key) {
    using U = typename Ordered<K>::U;
    const U u = __builtin_bit_cast(U, key);
    return u & Ordered<K>::kSign ? ~u : u | Ordered<K>::kSign;
}
template <typename K>
__device__ __forceinline__ K key_at(typename Ordered<K>::U order) {
    using U = typename Ordered<K>::U;
    return __builtin_bit_cast(K, order & Ordered<K>::kSign ? (U)(order & ~Ordered<K>::kSign) : (U)~order);
}

// Where a lane's register r stands in the row: registers are read C at a time, 64 lanes side by side.
template <int R, int WAVES>
struct Layout {
    static constexpr int C = R < 8 ? R : 8;
    static constexpr int kIds = 64 * R * WAVES;
    __device__ __forceinline__ static uint32_t id(int r) {
        const uint32_t thread = threadIdx.x & (64 * WAVES - 1);
        return ((uint32_t)(r / C) * (64 * WAVES) + thread) * C + r % C;
    }
};

// The row's values, `fill` beyond its end.
template <int R, int WAVES, typename T>
__device__ __forceinline__ void read_row(const T* __restrict__ row, uint32_t n, float fill, float (&v)[R]) {
    using L = Layout<R, WAVES>;
#pragma unroll
    for (int q = 0; q < R / L::C; ++q) {
        const uint32_t first = L::id(q * L::C);
        float part[L::C];
        if (first + L::C <= n) {
            load_n<L::C>(row + first, part);
        } else {
#pragma unroll
            for (int j = 0; j < L::C; ++j) part[j] = first + j < n ? to_f32(row[first + j]) : fill;
        }
#pragma unroll
        for (int j = 0; j < L::C; ++j) v[q * L::C + j] = part[j];
    }
}

// Selects the k largest keys > -inf, the lowest places first among equal ones: won has bit r for register r.
// Places ascend with the chunk r / C, then the thread, then r % C.  Returns how many were selected.
template <int R, int C, int WAVES, typename K>
__device__ __forceinline__ uint32_t select_largest(const K (&key)[R], uint32_t k, Meet<WAVES>& meet, uint32_t& won) {
    using U = typename Ordered<K>::U;
    const auto count = [&](K least) {
        uint32_t c = 0;
#pragma unroll
        for (int r = 0; r < R; ++r) c += (uint32_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64(key[r] >= least));
        return meet.total(c);
    };
    K top = key[0];
#pragma unroll
    for (int r = 1; r < R; ++r) top = max_of(top, key[r]);
    const K largest = meet.max(top);
    won = 0;
    uint32_t live = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) live += (uint32_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64(key[r] > (K)-INFINITY));
    live = meet.total(live);
    if (live <= k) {
#pragma unroll
        for (int r = 0; r < R; ++r) won |= key[r] > (K)-INFINITY ? 1u << r : 0u;
        return live;
    }
    U lo = order_of((K)-INFINITY), hi = order_of(largest) + 1;   // at least k keys are >= lo, fewer than k >= hi
    if (k <= 64 * WAVES) lo = order_of(-meet.max(-top));
    bool exact = false;
    while (hi - lo > 1) {
        const U mid = lo + (hi - lo) / 2;
        const uint32_t c = count(key_at<K>(mid));
        if (c >= k) lo = mid;
        else hi = mid;
        if (c == k) {
            exact = true;
            break;
        }
    }
    const K least = key_at<K>(lo);
#pragma unroll
    for (int r = 0; r < R; ++r) won |= key[r] >= least ? 1u << r : 0u;
    if (exact) return k;
    // `least` is a key: what lies above it wins, and the first of those equal to it
    uint32_t above = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) above += (uint32_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64(key[r] > least));
    uint32_t room = k - meet.total(above);
    const uint32_t lane = threadIdx.x & 63, wave = WAVES > 1 ? threadIdx.x >> 6 : 0;
#pragma unroll
    for (int q = 0; q < R / C; ++q) {
        uint32_t before = 0, here = 0;   // equal keys of this chunk: in the lanes below, and in the wave
#pragma unroll
        for (int j = 0; j < C; ++j) {
            const unsigned long long eq = __builtin_amdgcn_ballot_w64(key[q * C + j] == least);
            before += (uint32_t)__builtin_popcountll(eq & ((1ull << lane) - 1ull));
            here += (uint32_t)__builtin_popcountll(eq);
        }
        if constexpr (WAVES > 1) {
            double* s = meet.slot + (meet.turn++ & 1) * WAVES;
            if (lane == 0) s[wave] = (double)here;
            __syncthreads();
            here = 0;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                before += (uint32_t)w < wave ? (uint32_t)s[w] : 0u;
                here += (uint32_t)s[w];
            }
        }
#pragma unroll
        for (int j = 0; j < C; ++j)
            if (key[q * C + j] == least) {
                if (before >= room) won &= ~(1u << (q * C + j));
                ++before;
            }
        room -= here < room ? here : room;
    }
    return k;
}

// v_exp_f32 and v_rcp_f32 are within a step of their value; arguments are rounded once more on the way to base 2
__device__ __forceinline__ float exp_fast(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }
__device__ __forceinline__ float rcp_fast(float x) { return __builtin_amdgcn_rcpf(x); }
// x - m for an exponential whose largest argument is m: infinities of the same sign differ by nothing
template <typename K>
__device__ __forceinline__ K below(K x, K m) {
    return x == m ? (K)0 : x - m;
}
__device__ __forceinline__ float sigmoid(float x) { return rcp_fast(1.0f + exp_fast(-x)); }
// e^x in binary64: x = n ln 2 + r with |r| <= ln 2 / 2, the Taylor polynomial of degree 13 in r (its first missing term is
// below 2^-57), scaled by 2^n.  Within two steps of its value; arguments beyond +-800 give infinity and 0.
__device__ __forceinline__ double exp64(double x) {
    x = fmin(fmax(x, -800.0), 800.0);
    const double n = rint(x * 1.44269504088896340736);
    double r = fma(n, -6.93147180369123816490e-01, x);   // ln 2 in two parts, the first short enough that n times it is exact
    r = fma(n, -1.90821492927058770002e-10, r);
    double p = 1.0 / 6227020800.0;
    p = fma(p, r, 1.0 / 479001600.0);
    p = fma(p, r, 1.0 / 39916800.0);
    p = fma(p, r, 1.0 / 3628800.0);
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return ldexp(p, (int)n);
}
// 1 / x for 1 <= x < 1e305: the hardware's approximation and two Newton steps
__device__ __forceinline__ double rcp64(double x) {
    double y = __builtin_amdgcn_rcp(x);
    y = fma(y, fma(-x, y, 1.0), y);
    return fma(y, fma(-x, y, 1.0), y);
}
__device__ __forceinline__ double sigmoid(double x) { return rcp64(1.0 + exp64(fmin(fmax(-x, -700.0), 700.0))); }
// sigmoid(x) e^-c, c <= 0 no smaller than any x that is negative: ratios of sigmoids that would all underflow
__device__ __forceinline__ float sigmoid_over(float x, float c) {
    const float t = rcp_fast(1.0f + exp_fast(-fabsf(x)));
    return x < 0.0f ? exp_fast(below(x, c)) * t : t;
}

__device__ __forceinline__ uint32_t bits_in(unsigned long long mask) { return (uint32_t)__builtin_popcountll(mask); }

// inclusive sums over the lanes of a wave
__device__ __forceinline__ uint32_t scan_lanes(uint32_t v) {
    v += (uint32_t)dpp<0x111, 0xF>(0, (int)v);   // one lane up in a row of 16, two, four, eight
    v += (uint32_t)dpp<0x112, 0xF>(0, (int)v);
    v += (uint32_t)dpp<0x114, 0xF>(0, (int)v);
    v += (uint32_t)dpp<0x118, 0xF>(0, (int)v);
    v += (uint32_t)dpp<0x142, 0xA>(0, (int)v);
    v += (uint32_t)dpp<0x143, 0xC>(0, (int)v);
    return v;
}

// here[q]: what this thread holds in chunk q (at most 8).  place[q]: what stands before it, chunks first, then threads; returns
// the total.
template <int Q, int WAVES>
__device__ __forceinline__ uint32_t places(const uint32_t (&here)[Q], uint32_t (&place)[Q], uint32_t* starts) {
    uint32_t total = 0, packed[(Q + 1) / 2], sums[(Q + 1) / 2];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int p = 0; p < (Q + 1) / 2; ++p) {
        packed[p] = here[2 * p] | (2 * p + 1 < Q ? here[2 * p + 1] << 16 : 0u);
        sums[p] = scan_lanes(packed[p]);
    }
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const uint32_t in_wave = ((uint32_t)last_lane((int)sums[q / 2]) >> (q % 2 * 16)) & 0xFFFFu;
        place[q] = ((sums[q / 2] - packed[q / 2]) >> (q % 2 * 16)) & 0xFFFFu;
        if constexpr (WAVES == 1) {
            place[q] += total;
            total += in_wave;
        } else {
            if (lane == 0) starts[q * WAVES + wave] = in_wave;
        }
    }
    if constexpr (WAVES > 1) {
        __syncthreads();
        uint32_t at = 0;
#pragma unroll
        for (int q = 0; q < Q; ++q)
            for (int w = 0; w < WAVES; ++w) {
                if ((uint32_t)w == wave) place[q] += at;
                at += starts[q * WAVES + w];
            }
        total = at;
        __syncthreads();
    }
    return total;
}

struct WinnersArgs {
    sdrb_winners_spec w;
    uint64_t n_rows, ld;
    uint32_t n_ids;
    uint32_t group_size, group_lanes_log2;   // ids of a group; lanes that look at one group together
    uint32_t group_magic;                    // id * group_magic >> 31 is the id's group
    uint32_t lds_row;                        // bytes of dynamic LDS a row has
};

// candidates a thread takes at most; the threshold is looked for where k is at most this part of the lanes
constexpr int kHeld = 4;
constexpr uint32_t kLanePart = 48;

// A row of scores in its threads' registers, and the steps that choose its winners.  SHARES: keys are shares (+ bias), exactly
// so in binary64; else the scores.
template <int R, int WAVES, bool SHARES, typename T>
struct Row {
    using L = Layout<R, WAVES>;
    using K = std::conditional_t<SHARES, double, float>;
    static constexpr int C = L::C, Q = R / C;

    const WinnersArgs& a;
    const T* s_row;
    unsigned char* mine;    // LDS of the row
    uint32_t* starts;       // LDS, [WAVES][at most 8] where WAVES > 1
    Meet<WAVES> meet;
    float s[R];
    float top, inv_sum;     // of a softmax over the row

    __device__ __forceinline__ bool sig() const { return a.w.score == SDRB_SCORE_SIGMOID; }
    __device__ __forceinline__ uint32_t thread() const { return WAVES == 1 ? threadIdx.x & 63 : threadIdx.x; }
    // the winners in LDS, ascending
    __device__ __forceinline__ int32_t* win_ids() const { return reinterpret_cast<int32_t*>(mine); }
    __device__ __forceinline__ float* win_scores() const { return reinterpret_cast<float*>(mine) + a.w.k; }
    __device__ __forceinline__ void sync() const {   // LDS written by this row's waves before, read after
        if constexpr (WAVES == 1) {
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        } else {
            __syncthreads();
        }
    }

    // 1 / sum of the row's exponentials, which every share of a softmax has as a factor
    __device__ __forceinline__ double exact_inverse_sum() {
        double sum = 0.0;
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (s[r] > -INFINITY) sum += exp64(below((double)s[r], (double)top));
        return 1.0 / meet.sum(sum);
    }
    __device__ __forceinline__ double exact_key(float x, uint32_t id, double inverse_sum) const {
        double key = sig() ? sigmoid((double)x) : exp64(below((double)x, (double)top)) * inverse_sum;
        if (a.w.bias) key += (double)a.w.bias[id];
        return x > -INFINITY && key > -INFINITY ? key : -INFINITY;   // (a NaN of the bias is no key)
    }

    // keys of the kept groups stay; false where `slack` > 0 and binary32 keys do not tell the groups apart.  slack: how far
    // a key may be off, beside its own rounding
    template <typename F>
    __device__ __forceinline__ bool keep_groups(F (&key)[R], F slack) {
        const sdrb_winners_spec& w = a.w;
        F* keys = reinterpret_cast<F*>(mine);
        F* group = keys + a.n_ids;                                          // [groups]
        uint32_t* kept = reinterpret_cast<uint32_t*>(group + w.groups);     // a bit a group
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (L::id(r) < a.n_ids) keys[L::id(r)] = key[r];
        sync();
        // a group's one or two largest keys, by 2^group_lanes_log2 threads a group
        const uint32_t lanes = 1u << a.group_lanes_log2, lane = threadIdx.x & 63;
        F size = (F)0;   // of the keys that are summed
        for (uint32_t g0 = 0; g0 < w.groups; g0 += (64 * WAVES) >> a.group_lanes_log2) {
            const uint32_t g = g0 + (thread() >> a.group_lanes_log2);
            F best = (F)-INFINITY, next = (F)-INFINITY;
            if (g < w.groups)
                for (uint32_t e = thread() & (lanes - 1); e < a.group_size; e += lanes) {
                    const F k = keys[g * a.group_size + e];
                    next = k > best ? best : (k > next ? k : next);
                    best = max_of(best, k);
                }
            for (uint32_t d = 1; d < lanes; d <<= 1) {
                const F b = __shfl_xor(best, (int)d, 64), n = __shfl_xor(next, (int)d, 64);
                next = b > best ? max_of(best, n) : max_of(next, b);
                best = max_of(best, b);
            }
            const bool two = w.group_top > 1 && next > (F)-INFINITY;
            if (g < w.groups && (thread() & (lanes - 1)) == 0) group[g] = two ? best + next : best;
            if (best > (F)-INFINITY) size = max_of(size, (best < 0 ? -best : best) + (two ? (next < 0 ? -next : next) : (F)0));
        }
        sync();
        bool sure = true;
        if (slack > (F)0) size = meet.max(size);
        if (WAVES == 1 || threadIdx.x < 64) {
            // a group is kept if fewer than top_groups groups stand before it; thread lane + 64 j looks at one each
            F worst = (F)INFINITY, lost = (F)-INFINITY;
            for (uint32_t g0 = 0; g0 < w.groups; g0 += 64) {
                const uint32_t g = g0 + lane;
                const F mine_is = g < w.groups ? group[g] : (F)-INFINITY;
                uint32_t before = 0;
                for (uint32_t o = 0; o < w.groups; ++o) {
                    const F other = group[o];
                    before += other > mine_is || (other == mine_is && o < g) ? 1u : 0u;
                }
                const bool in = mine_is > (F)-INFINITY && before < w.top_groups;
                const unsigned long long m = __builtin_amdgcn_ballot_w64(in);
                if (lane == 0) {
                    kept[g0 / 32] = (uint32_t)m;
                    kept[g0 / 32 + 1] = (uint32_t)(m >> 32);
                }
                if (in) worst = mine_is < worst ? mine_is : worst;
                else lost = max_of(lost, mine_is);
            }
            if (slack > (F)0) {
                worst = -wave_reduce(-worst, (F)-INFINITY, max_of<F>);
                lost = wave_reduce(lost, (F)-INFINITY, max_of<F>);
                // two sums, of two keys each: every one off by slack and three roundings of at most `size`
                if (lost > (F)-INFINITY && !(worst - lost > 4 * slack + size * (F)0x1p-20)) sure = false;
            }
        }
        if (WAVES > 1 && slack > (F)0) sure = meet.total(threadIdx.x < 64 && !sure ? 1u : 0u) == 0;
        sync();
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const uint32_t g = __umulhi(2 * L::id(r), a.group_magic);   // (ids beyond the row have no key)
            if (key[r] > (F)-INFINITY && !(kept[g >> 5] >> (g & 31) & 1u)) key[r] = (F)-INFINITY;
        }
        sync();
        return sure;
    }

    // the winners among keys that the threads hold C at a time, to LDS
    template <int H, int CH, typename F, typename G>
    __device__ __forceinline__ uint32_t put_winners(const K (&key)[H], F id_of, G score_of) {
        uint32_t won, here[H / CH], place[H / CH];
        const uint32_t found = select_largest<H, CH, WAVES>(key, a.w.k, meet, won);
#pragma unroll
        for (int q = 0; q < H / CH; ++q) here[q] = __popc((won >> (q * CH)) & (uint32_t)((1ull << CH) - 1));
        places<H / CH, WAVES>(here, place, starts);
#pragma unroll
        for (int j = 0; j < H; ++j)
            if ((won >> j) & 1u) {
                win_ids()[place[j / CH]] = id_of(j);
                win_scores()[place[j / CH]++] = score_of(j);
            }
        sync();
        return found;
    }

    // the candidates that a threshold leaves, and the winners among them; false where the row needs choose_among_all
    __device__ __forceinline__ bool choose_among_candidates(uint32_t& found) {
        const sdrb_winners_spec& w = a.w;
        if (w.k > kLanePart * WAVES) return false;
        float rough[R], slack = 0.0f;
        if constexpr (SHARES) {
            // Off by less than 3.1 * 2^-24 for the sigmoid -- 1.5 |x| + 2 steps in its exponential t, which enter the result
            // with t / (1 + t)^2, and two roundings -- and than 2^-17 of the largest share for the softmax, 67 * 2^-24 by its
            // own exponential and a sum of at most 32 + 6 + 8 additions.
            slack = sig() ? 0x1p-22f : inv_sum * 0x1p-17f;
#pragma unroll
            for (int r = 0; r < R; ++r) rough[r] = sig() ? sigmoid(s[r]) : exp_fast(below(s[r], top)) * inv_sum;
            if (w.bias) {
                float b[R];
                read_row<R, WAVES>(w.bias, a.n_ids, 0.0f, b);
#pragma unroll
                for (int r = 0; r < R; ++r) rough[r] += b[r];
            }
#pragma unroll
            for (int r = 0; r < R; ++r) rough[r] = s[r] > -INFINITY && rough[r] > -INFINITY ? rough[r] : -INFINITY;
        } else {
#pragma unroll
            for (int r = 0; r < R; ++r) rough[r] = s[r];
        }
        if (w.groups > 1 && !keep_groups<float>(rough, slack)) return false;

        float mine_top = rough[0];
#pragma unroll
        for (int r = 1; r < R; ++r) mine_top = max_of(mine_top, rough[r]);
        const auto reach = [&](float t) { return meet.total(bits_in(__builtin_amdgcn_ballot_w64(mine_top >= t))); };
        float t = -INFINITY;
        if (meet.total(bits_in(__builtin_amdgcn_ballot_w64(mine_top > -INFINITY))) >= w.k) {
            const float least = -meet.max(mine_top > -INFINITY ? -mine_top : -INFINITY);   // of the live lanes
            uint32_t lo = order_of(least), hi = order_of(meet.max(mine_top)) + 1;
            const uint32_t enough = w.k + w.k / 8 + 1;
            while (hi - lo > 1) {
                const uint32_t mid = lo + (hi - lo) / 2, c = reach(key_at<float>(mid));
                if (c >= w.k) lo = mid;
                else hi = mid;
                if (c >= w.k && c <= enough) break;
            }
            t = key_at<float>(lo);
            // k keys are no smaller than t less what a key can be off; a key as large may seem smaller by as much again
            if (SHARES) t -= 2.0f * slack + fabsf(t) * 0x1p-21f;   // (an infinite t becomes NaN, which nothing reaches)
        }
        uint32_t bits = 0, here[Q], place[Q];
#pragma unroll
        for (int r = 0; r < R; ++r) bits |= rough[r] >= t && rough[r] > -INFINITY ? 1u << r : 0u;
#pragma unroll
        for (int q = 0; q < Q; ++q) here[q] = __popc((bits >> (q * C)) & ((1u << C) - 1u));
        const uint32_t n = places<Q, WAVES>(here, place, starts);
        if (n > 64u * WAVES * kHeld || (n < w.k && t != -INFINITY)) return false;
        int32_t* list = reinterpret_cast<int32_t*>(mine);
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            uint32_t b = (bits >> (q * C)) & ((1u << C) - 1u), at = place[q];
            while (b) {
                list[at++] = (int32_t)(L::id(q * C) + (uint32_t)__builtin_ctz(b));
                b &= b - 1;
            }
        }
        sync();
        found = n <= 64 * WAVES ? choose_from_list<1>(list, n) : choose_from_list<kHeld>(list, n);
        return true;
    }
    template <int H>
    __device__ __forceinline__ uint32_t choose_from_list(const int32_t* list, uint32_t n) {
        K key[H];
        float x[H];
        int32_t id[H];
        const double inverse_sum = SHARES && !sig() ? exact_inverse_sum() : 0.0;
#pragma unroll
        for (int j = 0; j < H; ++j) {
            const uint32_t i = j * 64 * WAVES + thread();
            key[j] = (K)-INFINITY;
            x[j] = -INFINITY;
            id[j] = -1;
            if (i < n) {
                id[j] = list[i];
                x[j] = to_f32(s_row[id[j]]) + 0.0f;   // -0 is 0
                if constexpr (SHARES) key[j] = exact_key(x[j], (uint32_t)id[j], inverse_sum);
                else key[j] = x[j];
            }
        }
        return put_winners<H, 1>(key, [&](int j) { return id[j]; }, [&](int j) { return x[j]; });
    }

    // bisection over all keys
    __device__ __forceinline__ uint32_t choose_among_all() {
        K key[R];
        const double inverse_sum = SHARES && !sig() ? exact_inverse_sum() : 0.0;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if constexpr (SHARES) key[r] = L::id(r) < a.n_ids ? exact_key(s[r], L::id(r), inverse_sum) : -INFINITY;
            else key[r] = s[r];
        }
        if (a.w.groups > 1) keep_groups<K>(key, (K)0);
        return put_winners<R, C>(key, [&](int r) { return (int32_t)L::id(r); }, [&](int r) { return s[r]; });
    }
};

template <int R, int WAVES, bool SHARES, typename T>
__global__ __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES) void k_winners(WinnersArgs a, const T* __restrict__ scores,
                                                                           int32_t* __restrict__ out_ids,
                                                                           float* __restrict__ out_weights) {
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    __shared__ double slots[2 * WAVES];
    __shared__ uint32_t starts[WAVES == 1 ? 1 : WAVES * 8];
    const uint32_t wave = threadIdx.x >> 6;
    const uint64_t row = WAVES == 1 ? (uint64_t)blockIdx.x * 4 + wave : blockIdx.x;
    if (row >= a.n_rows) return;
    const sdrb_winners_spec& w = a.w;
    Row<R, WAVES, SHARES, T> x{a, scores + row * a.ld, lds + (WAVES == 1 ? wave * a.lds_row : 0u), starts, {slots, 0}, {}, 0.0f, 0.0f};
    const bool sig = x.sig();
    read_row<R, WAVES>(x.s_row, a.n_ids, -INFINITY, x.s);
#pragma unroll
    for (int r = 0; r < R; ++r) x.s[r] = x.s[r] > -INFINITY ? x.s[r] + 0.0f : -INFINITY;   // NaN is no score; -0 is 0
    if (!sig && (SHARES || !w.renormalise)) {   // a softmax over the row
        float m = x.s[0], sum = 0.0f;
#pragma unroll
        for (int r = 1; r < R; ++r) m = max_of(m, x.s[r]);
        x.top = x.meet.max(m);
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (x.s[r] > -INFINITY) sum += exp_fast(below(x.s[r], x.top));
        x.inv_sum = rcp_fast(x.meet.sum(sum));
    }
    uint32_t found;
    if (!x.choose_among_candidates(found)) {
        x.sync();
        found = x.choose_among_all();
    }

    // the weights, a winner a thread
    const uint32_t thread = x.thread();
    const int32_t* win_id = x.win_ids();
    const float* win_s = x.win_scores();
    float shift = 0.0f, norm = w.scale;
    if (w.renormalise) {
        float m = -INFINITY;
        for (uint32_t i = thread; i < found; i += 64 * WAVES) m = max_of(m, win_s[i]);
        shift = x.meet.max(m);
        if (sig) shift = shift < 0.0f ? shift : 0.0f;
        float sum = 0.0f;
        for (uint32_t i = thread; i < found; i += 64 * WAVES) sum += sig ? sigmoid_over(win_s[i], shift) : exp_fast(below(win_s[i], shift));
        norm = w.scale * rcp_fast(x.meet.sum(sum));
    }
    int32_t* ids = out_ids + row * w.k;
    float* weights = out_weights + row * w.k;
    for (uint32_t i = thread; i < w.k; i += 64 * WAVES) {
        int32_t id = -1;
        float weight = 0.0f;
        if (i < found) {
            id = win_id[i];
            const float v = win_s[i];
            if (sig) weight = norm * (w.renormalise ? sigmoid_over(v, shift) : sigmoid(v));
            else weight = norm * (w.renormalise ? exp_fast(below(v, shift)) : exp_fast(below(v, x.top)) * x.inv_sum);
        }
        ids[i] = id;
        weights[i] = weight;
    }
}

struct WinnersGradArgs {
    sdrb_winners_spec w;
    uint64_t n_rows, ld, out_ld;
    uint32_t n_ids;
    uint32_t lds_row;
};

// d scores of a row, from its winners and their weights' gradient, laid out in LDS: a row of zeros into which the winners'
// values are put.  Only a softmax over the whole row reads the row; the other gradients read the winners' scores alone.
// Bound: the write of the result.
template <int R, int WAVES, bool WHOLE, typename T, typename O>
__global__ __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES) void k_winners_grad(WinnersGradArgs a, const T* __restrict__ scores,
                                                                                const int32_t* __restrict__ ids_in,
                                                                                const float* __restrict__ grad_in,
                                                                                O* __restrict__ out) {
    using L = Layout<R, WAVES>;
    constexpr int C = L::C;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    __shared__ double slots[2 * WAVES];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint64_t row = WAVES == 1 ? (uint64_t)blockIdx.x * 4 + wave : blockIdx.x;
    if (row >= a.n_rows) return;
    float* line = reinterpret_cast<float*>(lds + (WAVES == 1 ? wave * a.lds_row : 0u));   // [L::kIds]
    Meet<WAVES> meet{slots, 0};
    const auto sync = [] {
        if constexpr (WAVES == 1) {
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        } else {
            __syncthreads();
        }
    };
    const uint32_t thread = WAVES == 1 ? lane : threadIdx.x;
    const T* s_row = scores + row * a.ld;
    const int32_t* ids = ids_in + row * a.w.k;
    const float* grad = grad_in + row * a.w.k;
    const sdrb_winners_spec& w = a.w;
    const bool sig = w.score == SDRB_SCORE_SIGMOID;
    float s[WHOLE ? R : 1];
    if constexpr (WHOLE) read_row<R, WAVES>(s_row, a.n_ids, -INFINITY, s);
    const float zeros[C] = {};
#pragma unroll
    for (int q = 0; q < R / C; ++q) store_n<C>(line + L::id(q * C), zeros);
    sync();
    // a thread's winners: the score of place i, -inf where it holds none
    const auto score_at = [&](uint32_t i, int32_t& id) {
        id = ids[i];
        if (id < 0 || (uint32_t)id >= a.n_ids) return -INFINITY;
        const float x = to_f32(s_row[id]);
        return x > -INFINITY ? x : -INFINITY;   // (a NaN never won)
    };
    if constexpr (WHOLE) {
        for (uint32_t i = thread; i < w.k; i += 64 * WAVES) {
            int32_t id;
            if (score_at(i, id) > -INFINITY) line[id] = grad[i];
        }
        sync();
        float m = -INFINITY;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            s[r] = s[r] > -INFINITY ? s[r] : -INFINITY;   // (a NaN has no share)
            m = max_of(m, s[r]);
        }
        m = meet.max(m);
        float g[R], sum = 0.0f, dot = 0.0f;
#pragma unroll
        for (int q = 0; q < R / C; ++q) {
            float part[C];
            load_n<C>(line + L::id(q * C), part);
#pragma unroll
            for (int j = 0; j < C; ++j) g[q * C + j] = part[j];
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            s[r] = s[r] > -INFINITY ? exp_fast(below(s[r], m)) : 0.0f;
            sum += s[r];
            dot = fmaf(s[r], g[r], dot);
        }
        const float inv = rcp_fast(meet.sum(sum));
        dot = meet.sum(dot) * inv;
        const float scale = w.scale * inv;
#pragma unroll
        for (int r = 0; r < R; ++r) s[r] = s[r] > 0.0f ? scale * s[r] * (g[r] - dot) : 0.0f;
#pragma unroll
        for (int q = 0; q < R / C; ++q) {
            const uint32_t first = L::id(q * C);
            O* to = out + row * a.out_ld + first;
            if (first + C <= a.n_ids) {
                float part[C];
#pragma unroll
                for (int j = 0; j < C; ++j) part[j] = s[q * C + j];
                store_n<C>(to, part);
            } else {
#pragma unroll
                for (int j = 0; j < C; ++j)
                    if (first + j < a.n_ids) to[j] = from_f32<O>(s[q * C + j]);
            }
        }
    } else {
        float shift = 0.0f, inv = 1.0f, dot = 0.0f;
        const auto part_of = [&](float x) { return sig ? sigmoid_over(x, shift) : exp_fast(below(x, shift)); };
        if (w.renormalise) {
            float m = -INFINITY, sum = 0.0f;
            int32_t id;
            for (uint32_t i = thread; i < w.k; i += 64 * WAVES) m = max_of(m, score_at(i, id));
            shift = meet.max(m);
            if (sig) shift = shift < 0.0f ? shift : 0.0f;
            for (uint32_t i = thread; i < w.k; i += 64 * WAVES) {
                const float x = score_at(i, id);
                if (x > -INFINITY) {
                    const float p = part_of(x);
                    sum += p;
                    dot = fmaf(p, grad[i], dot);
                }
            }
            inv = rcp_fast(meet.sum(sum));
            dot = meet.sum(dot) * inv;
        }
        for (uint32_t i = thread; i < w.k; i += 64 * WAVES) {
            int32_t id;
            const float x = score_at(i, id);
            if (x > -INFINITY) {
                float d = w.renormalise ? part_of(x) * inv * (grad[i] - dot) : grad[i] * sigmoid(x);
                if (sig) d *= sigmoid(-x);
                line[id] = w.scale * d;
            }
        }
        sync();
        constexpr int V = 16 / sizeof(O);   // 16 bytes of the result a lane
        for (uint32_t first = thread * V; first < a.n_ids; first += 64 * WAVES * V) {
            float part[V];
            load_n<V>(line + first, part);
            O* to = out + row * a.out_ld + first;
            if (first + V <= a.n_ids) {
                store_n<V>(to, part);
            } else {
                for (int j = 0; j < V; ++j)
                    if (first + j < a.n_ids) to[j] = from_f32<O>(part[j]);
            }
        }
    }
}

// calls f(R, WAVES) with the smallest layout that holds n ids
template <typename F>
int with_layout(uint32_t n, F&& f) {
    using std::integral_constant;
    const auto one = integral_constant<int, 1>{};
    const auto eight = integral_constant<int, 8>{};
    if (n <= 64) return f(integral_constant<int, 1>{}, one);
    if (n <= 128) return f(integral_constant<int, 2>{}, one);
    if (n <= 256) return f(integral_constant<int, 4>{}, one);
    if (n <= 512) return f(integral_constant<int, 8>{}, one);
    if (n <= 1024) return f(integral_constant<int, 16>{}, one);
    if (n <= 2048) return f(integral_constant<int, 32>{}, one);
    if (n <= 4096) return f(integral_constant<int, 8>{}, eight);
    if (n <= 8192) return f(integral_constant<int, 16>{}, eight);
    return f(integral_constant<int, 32>{}, eight);
}

// more than 64 KiB of dynamic LDS has to be asked for
template <typename F>
int allow_lds(F* kernel, size_t bytes) {
    if (bytes > 65536) SDRB_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    return SDRB_OK;
}

}  // namespace

int launch_winners(const sdrb_dense& scores, const sdrb_winners_spec& spec, int32_t* ids, float* weights, hipStream_t stream) {
    WinnersArgs a{};
    a.w = spec;
    a.n_rows = scores.n_rows;
    a.ld = scores.ld;
    a.n_ids = (uint32_t)scores.n_cols;
    a.group_size = a.n_ids / spec.groups;
    a.group_magic = ((1u << 31) + a.group_size - 1) / a.group_size;   // exact for ids below 2^17
    const bool shares = spec.bias || (spec.groups > 1 && spec.group_top > 1);
    return with_layout(a.n_ids, [&](auto r, auto waves) {
        constexpr int R = decltype(r)::value, WAVES = decltype(waves)::value;
        a.group_lanes_log2 = 0;
        while (a.group_lanes_log2 < 6 && (spec.groups << (a.group_lanes_log2 + 1)) <= 64u * WAVES) ++a.group_lanes_log2;
        return with_type(scores.type, [&](auto t) {
            using T = decltype(t);
            const auto go = [&](auto s) {
                constexpr bool SHARES = decltype(s)::value;
                const size_t of_key = SHARES ? sizeof(double) : sizeof(float);
                const size_t grouped = spec.groups > 1 ? (a.n_ids + spec.groups) * of_key + kWinnersMaxGroups / 8 : 0;
                const size_t held = (a.n_ids < 64u * WAVES * kHeld ? a.n_ids : 64u * WAVES * kHeld) * sizeof(int32_t);
                const size_t listed = spec.k * 8 > held ? spec.k * 8 : held;
                a.lds_row = (uint32_t)(((grouped > listed ? grouped : listed) + 15) / 16 * 16);
                const size_t lds = (size_t)a.lds_row * (WAVES == 1 ? 4 : 1);
                const uint64_t blocks = WAVES == 1 ? (a.n_rows + 3) / 4 : a.n_rows;
                if (const int rc = allow_lds(&k_winners<R, WAVES, SHARES, T>, lds)) return rc;
                hipLaunchKernelGGL((k_winners<R, WAVES, SHARES, T>), dim3((uint32_t)blocks), dim3(WAVES == 1 ? 256 : 64 * WAVES), lds,
                                   stream, a, static_cast<const T*>(scores.data), ids, weights);
                SDRB_HIP(hipGetLastError());
                return SDRB_OK;
            };
            return shares ? go(std::true_type{}) : go(std::false_type{});
        });
    });
}

int launch_winners_grad(const sdrb_dense& scores, const sdrb_winners_spec& spec, const int32_t* ids, const float* grad_weights,
                        const sdrb_dense& out, hipStream_t stream) {
    WinnersGradArgs a{};
    a.w = spec;
    a.n_rows = scores.n_rows;
    a.ld = scores.ld;
    a.out_ld = out.ld;
    a.n_ids = (uint32_t)scores.n_cols;
    const bool whole = spec.score == SDRB_SCORE_SOFTMAX && !spec.renormalise;
    return with_layout(a.n_ids, [&](auto r, auto waves) {
        constexpr int R = decltype(r)::value, WAVES = decltype(waves)::value;
        a.lds_row = (uint32_t)(Layout<R, WAVES>::kIds + 8) * sizeof(float);   // (16 bytes of result are read at a time)
        const size_t lds = (size_t)a.lds_row * (WAVES == 1 ? 4 : 1);
        const uint64_t blocks = WAVES == 1 ? (a.n_rows + 3) / 4 : a.n_rows;
        return with_type(scores.type, [&](auto t) {
            return with_type(out.type, [&](auto o) {
                using T = decltype(t);
                using O = decltype(o);
                const auto go = [&](auto all) {
                    constexpr bool WHOLE = decltype(all)::value;
                    if (const int rc = allow_lds(&k_winners_grad<R, WAVES, WHOLE, T, O>, lds)) return rc;
                    hipLaunchKernelGGL((k_winners_grad<R, WAVES, WHOLE, T, O>), dim3((uint32_t)blocks), dim3(WAVES == 1 ? 256 : 64 * WAVES),
                                       lds, stream, a, static_cast<const T*>(scores.data), ids, grad_weights, static_cast<O*>(out.data));
                    SDRB_HIP(hipGetLastError());
                    return SDRB_OK;
                };
                return whole ? go(std::true_type{}) : go(std::false_type{});
            });
        });
    });
}

}  // namespace sdrb
