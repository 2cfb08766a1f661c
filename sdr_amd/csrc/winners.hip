// The k winners of every row of dense scores, with their weights, and the gradient of those weights to the scores.
//
// Shares: u = softmax of a row's live scores, or their sigmoids; a score of -inf or NaN is not live.  Keys: u + bias, or the
// scores where nothing is added to the shares (the same order).  A group's score is the sum of its one or two largest
// keys; the k largest keys inside the best groups win, ties go to the lowest group and id.
// Weights: scale * u, or, renormalised, scale * p with p = u / sum of the winners' u -- a softmax over the winners of
// l = s (softmax) or l = log sigmoid(s), which holds where every u underflows.
//
// A team of threads owns a row and holds its scores in registers, read once: 64 threads, two, four or eight times as many for
// more than 2048, 4096 and 8192 ids, or 16 where there are many short rows (four rows a wave: what a team does once, it does
// for four rows at a time).  Two steps choose the winners:
//  1. Candidates.  Of the threads' largest keys -- two a thread, each of half its registers -- a threshold is found that k of
//     them reach (a compare and a count a step), so at least k keys reach it, and few more: about 47 of 2048 for k = 40.  Keys
//     are binary32 here; where shares enter them the threshold is lowered by what their arithmetic can be off, so that no
//     winner is lost.
//  2. The candidates' ids go to LDS in ascending order, one a thread from there on; their keys are computed exactly, and the
//     k-th largest is found by bisection over the keys' order-preserving integers, which ends as soon as exactly k keys lie
//     at or above the middle.
// Shares that enter keys are computed in binary64 in the second step: whether an id wins hangs on the difference of two keys,
// which binary32 exponentials would decide by their own error.  Groups that binary32 does not tell apart are scored again
// exactly.  Rows whose candidates are too many -- large keys that few threads hold -- look for the threshold among all keys, and of
// equal keys take the lowest ids; where more keys than the list holds lie within an error of the threshold, the row is bisected by
// exact keys.  These are rolled loops that read the row anew: what runs rarely has to be short, since fetching instructions that no
// other wave has run costs more than running them (straight-line code of 900 instructions: 15 us).
// Bound: instruction issue, not memory: 8192 rows of 2048 bf16 scores, k = 40, in 14.7 us (34 MB read at 2.3 TB/s; 620 vector instructions
// a row, issued in 58 % of the CUs' busy time), 16384 rows of 256 in 8 groups, 4 of them taken, k = 8, in 15 to 18 us (17 MB; 320 a row, 74 %),
// 4096 rows of 16384, k = 328, in 124 us (134 MB); a single row of 256 in 4.9 us.  The gradients of 16384 rows of 128 and of 4099 rows of
// 2047 take 5.9 and 6.9 us (17 MB each).
#include <type_traits>

#include "dense_rows.h"

namespace sdrb {

namespace {

// ---- a wave's reductions ----
__device__ __forceinline__ uint32_t last_lane(uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, 63); }
__device__ __forceinline__ float last_lane(float v) { return __builtin_bit_cast(float, last_lane(__builtin_bit_cast(uint32_t, v))); }
__device__ __forceinline__ double last_lane(double v) {
    const uint64_t x = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, ((uint64_t)last_lane((uint32_t)(x >> 32)) << 32) | last_lane((uint32_t)x));
}
// op over the 64 lanes of a wave or each row of 16; `none` leaves every value as it is under op
template <int LANES, typename T, typename F>
__device__ __forceinline__ T lanes_reduce(T v, T none, F op) {
    v = op(v, dpp<0xB1, 0xF>(v, v));    // lanes 1 0 3 2
    v = op(v, dpp<0x4E, 0xF>(v, v));    // lanes 2 3 0 1
    v = op(v, dpp<0x141, 0xF>(v, v));   // the other half of 8
    v = op(v, dpp<0x140, 0xF>(v, v));   // the other half of 16
    if constexpr (LANES == 64) {
        v = op(v, dpp<0x142, 0xA>(none, v));   // lane 15 of the row of 16 below, into rows 1 and 3
        v = op(v, dpp<0x143, 0xC>(none, v));   // lane 31, into rows 2 and 3
        v = last_lane(v);
    }
    return v;
}
__device__ __forceinline__ uint32_t bits_in(unsigned long long mask) { return (uint32_t)__builtin_popcountll(mask); }
__device__ __forceinline__ uint32_t max_u32(uint32_t a, uint32_t b) { return a > b ? a : b; }
template <typename T>
__device__ __forceinline__ T max_of(T a, T b) {
    return a > b ? a : b;
}

// ---- keys as integers of the same order, above 0 for every key > -inf ----
__device__ __forceinline__ uint32_t order_of(float key) {
    const uint32_t u = __builtin_bit_cast(uint32_t, key);
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint64_t order_of(double key) {
    const uint64_t u = __builtin_bit_cast(uint64_t, key);
    return u ^ ((uint64_t)((int64_t)u >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ float key_at(uint32_t order) {
    return __builtin_bit_cast(float, order & 0x80000000u ? order & 0x7FFFFFFFu : ~order);
}
constexpr uint32_t kOrderOfNone = 0x007FFFFFu;   // of -inf
// Low bits of a score's order that its type leaves alike: a bisection stops short of them.
template <typename T>
constexpr int kAlike = std::is_same_v<T, bf16> ? 16 : std::is_same_v<T, f16> ? 13 : 0;

// ---- the threads of a row: 16 lanes, a wave, or up to eight waves that meet in LDS ----
template <int THREADS>
struct Team {
    static constexpr int kWaves = THREADS / 64;   // 0: a row of 16 lanes
    static constexpr int kLanes = THREADS < 64 ? THREADS : 64;
    double* slot;       // LDS, [2][kWaves] where kWaves > 1
    uint32_t* starts;   // LDS, [8][kWaves] where kWaves > 1
    uint32_t turn;

    __device__ __forceinline__ static uint32_t thread() { return threadIdx.x & (THREADS - 1); }
    __device__ __forceinline__ static uint32_t wave() { return threadIdx.x >> 6; }
    __device__ __forceinline__ static void sync() {   // LDS written by this row's threads before, read after
        if constexpr (kWaves > 1) {
            __syncthreads();
        } else {
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        }
    }
    template <typename T, typename F>
    __device__ __forceinline__ T over_waves(T v, F op) {   // v: the same in a wave
        if constexpr (kWaves > 1) {
            double* s = slot + (turn++ & 1) * kWaves;   // the turn before may still be read while this one is written
            if ((threadIdx.x & 63) == 0) s[wave()] = (double)v;
            __syncthreads();
            v = (T)s[0];
#pragma unroll
            for (int k = 1; k < kWaves; ++k) v = op(v, (T)s[k]);
        }
        return v;
    }
    template <typename T>
    __device__ __forceinline__ T sum(T v) {
        const auto add = [](T a, T b) { return a + b; };
        return over_waves(lanes_reduce<kLanes>(v, T(0), add), add);
    }
    __device__ __forceinline__ uint32_t max(uint32_t v) { return over_waves(lanes_reduce<kLanes>(v, 0u, max_u32), max_u32); }
    __device__ __forceinline__ uint32_t min(uint32_t v) { return ~max(~v); }
    __device__ __forceinline__ float max(float v) { return key_at(max(order_of(v))); }
    __device__ __forceinline__ double max(double v) {   // (of few calls: no integers here)
        return over_waves(lanes_reduce<kLanes>(v, (double)-INFINITY, max_of<double>), max_of<double>);
    }
    // this row's lanes of a ballot: a wave's, or 16 at the bottom
    __device__ __forceinline__ static unsigned long long own(unsigned long long ballot) {
        if constexpr (kWaves == 0) {
            const uint32_t half = threadIdx.x & 32 ? (uint32_t)(ballot >> 32) : (uint32_t)ballot;
            return __builtin_amdgcn_ubfe(half, threadIdx.x & 16, 16);
        }
        return ballot;
    }
    // threads of the row that say yes
    __device__ __forceinline__ uint32_t count(bool yes) {
        return over_waves(bits_in(own(__builtin_amdgcn_ballot_w64(yes))), [](uint32_t a, uint32_t b) { return a + b; });
    }
    // registers of the row's threads that say yes
    template <int R, typename F>
    __device__ __forceinline__ uint32_t count_all(F yes) {
        uint32_t c = 0;
        if constexpr (kWaves == 0 && R > 1) {
#pragma unroll
            for (int r = 0; r < R; ++r) c += yes(r) ? 1u : 0u;
            return sum(c);
        } else {
#pragma unroll
            for (int r = 0; r < R; ++r) c += bits_in(own(__builtin_amdgcn_ballot_w64(yes(r))));
            return over_waves(c, [](uint32_t a, uint32_t b) { return a + b; });
        }
    }
    // here[q]: what this thread holds in chunk q (at most 8).  place[q]: what stands before it, chunks first, then threads;
    // returns the total.
    template <int Q>
    __device__ __forceinline__ uint32_t places(const uint32_t (&here)[Q], uint32_t (&place)[Q]) {
        uint32_t total = 0, packed[(Q + 1) / 2], sums[(Q + 1) / 2], ends[(Q + 1) / 2];
#pragma unroll
        for (int p = 0; p < (Q + 1) / 2; ++p) {   // two chunks a register: at most 512 a wave in each
            packed[p] = here[2 * p] | (2 * p + 1 < Q ? here[2 * p + 1] << 16 : 0u);
            const uint32_t v = scan_lanes<kLanes>(packed[p]);
            if constexpr (kWaves == 0) ends[p] = dpp<0x15F, 0xF>(v, v);   // lane 15 of the row
            else ends[p] = last_lane(v);
            sums[p] = v;
        }
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            const uint32_t in_wave = (ends[q / 2] >> (q % 2 * 16)) & 0xFFFFu;
            place[q] = ((sums[q / 2] - packed[q / 2]) >> (q % 2 * 16)) & 0xFFFFu;
            if constexpr (kWaves > 1) {
                if ((threadIdx.x & 63) == 0) starts[q * kWaves + wave()] = in_wave;
            } else {
                place[q] += total;
                total += in_wave;
            }
        }
        if constexpr (kWaves > 1) {
            __syncthreads();
#pragma unroll
            for (int q = 0; q < Q; ++q)
                for (int w = 0; w < kWaves; ++w) {
                    if ((uint32_t)w == wave()) place[q] += total;
                    total += starts[q * kWaves + w];
                }
            __syncthreads();
        }
        return total;
    }
};

// Where a thread's register r stands in the row: registers are read C at a time, the row's threads side by side.
template <int R, int THREADS>
struct Layout {
    static constexpr int C = R < 8 ? R : 8;
    static constexpr int kIds = THREADS * R;
    __device__ __forceinline__ static uint32_t id(int r) {
        return ((uint32_t)(r / C) * THREADS + Team<THREADS>::thread()) * C + r % C;
    }
};

// The row's values, `fill` beyond its end.
template <int R, int THREADS, typename T>
__device__ __forceinline__ void read_row(const T* __restrict__ row, uint32_t n, float fill, float (&v)[R]) {
    using L = Layout<R, THREADS>;
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
// scores: a NaN is none (the maximum of it and -inf is -inf); -0 is 0
template <int R, int THREADS, typename T>
__device__ __forceinline__ void read_scores(const T* __restrict__ row, uint32_t n, float (&v)[R]) {
    read_row<R, THREADS>(row, n, -INFINITY, v);
#pragma unroll
    for (int r = 0; r < R; ++r) v[r] = fmaxf(v[r] + 0.0f, -INFINITY);
}

// Selects the k largest orders above `none`, the lowest places first among equal ones: won has bit r for register r.
// Places ascend with the chunk r / C, then the thread, then r % C.  Returns how many were selected.
template <int R, int C, int THREADS, typename U>
__device__ __forceinline__ uint32_t select_largest(const U (&key)[R], U none, uint32_t k, Team<THREADS>& team, uint32_t& won) {
    // the highest words decide where the bisection starts
    const auto high = [](U u) { return (uint32_t)(u >> (8 * sizeof(U) - 32)); };
    U top = key[0];
#pragma unroll
    for (int r = 1; r < R; ++r) top = max_of(top, key[r]);
    won = 0;
    const uint32_t live = team.template count_all<R>([&](int r) { return key[r] > none; });
    if (live <= k) {
#pragma unroll
        for (int r = 0; r < R; ++r) won |= key[r] > none ? 1u << r : 0u;
        return live;
    }
    // at least k keys are >= lo, fewer than k >= hi
    U hi = ((U)team.max(high(top)) << (8 * sizeof(U) - 32)) + ((U)1 << (8 * sizeof(U) - 32));
    U lo = none;
    if (k <= THREADS) lo = max_of(none, (U)team.min(high(top)) << (8 * sizeof(U) - 32));   // every thread has a key >= this
    uint32_t exact = 0;
    while (hi - lo > 1 && !exact) {
        const U mid = lo + (hi - lo) / 2;
        const uint32_t c = team.template count_all<R>([&](int r) { return key[r] >= mid; });
        if (c >= k) lo = mid;
        else hi = mid;
        exact = c == k;
    }
#pragma unroll
    for (int r = 0; r < R; ++r) won |= key[r] >= lo ? 1u << r : 0u;
    if (exact) return k;
    // `lo` is a key: what lies above it wins, and the first of those equal to it
    const uint32_t room = k - team.template count_all<R>([&](int r) { return key[r] > lo; });
    uint32_t here[R / C], place[R / C];
#pragma unroll
    for (int q = 0; q < R / C; ++q) {
        here[q] = 0;
#pragma unroll
        for (int j = 0; j < C; ++j) here[q] += key[q * C + j] == lo ? 1u : 0u;
    }
    team.places(here, place);
#pragma unroll
    for (int r = 0; r < R; ++r)
        if (key[r] == lo && place[r / C]++ >= room) won &= ~(1u << r);
    return k;
}

// The same for one key a lane of a row of 16: a key's rank is the number of keys before it, met by turning the row 15 times.
template <int N>
__device__ __forceinline__ uint32_t ranked_before(uint64_t key, uint32_t thread) {
    if constexpr (N == 0) {
        return 0;
    } else {
        const uint32_t lo = dpp<0x120 + N, 0xF>(0u, (uint32_t)key), hi = dpp<0x120 + N, 0xF>(0u, (uint32_t)(key >> 32));
        const uint64_t other = ((uint64_t)hi << 32) | lo;   // of the lane N below, or 16 - N above
        return ranked_before<N - 1>(key, thread) + (other > key || (other == key && thread >= (uint32_t)N) ? 1u : 0u);
    }
}

// v_exp_f32 and v_rcp_f32 are within a step of their value; arguments are rounded once more on the way to base 2, which costs 3 |x|
// half steps of the result: for approximate keys, and for sums over a row, where a small term's error is small beside the sum
__device__ __forceinline__ float exp_fast(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }
__device__ __forceinline__ float rcp_fast(float x) { return __builtin_amdgcn_rcpf(x); }
// x - m for an exponential whose largest argument is m: infinities of the same sign differ by nothing
template <typename K>
__device__ __forceinline__ K below(K x, K m) {
    return x == m ? (K)0 : x - m;
}
__device__ __forceinline__ float sigmoid_fast(float x) { return rcp_fast(1.0f + exp_fast(-x)); }
// e^(x - m) for x <= m, within 1.5 steps of its value however far x lies below m (0 below 2^-126): for weights and gradients.  What x - m and
// its product with log2 e lose to rounding is found exactly and put back as a factor 1 + r ln 2.
__device__ __forceinline__ float exp_over(float x, float m) {
    const float d = fmaxf(below(x, m), -150.0f), back = d - x;
    const float lost = d > -150.0f && x != m ? (x - (d - back)) - (m + back) : 0.0f;   // (x and m finite)
    const float t = d * 1.44269504088896341f;
    const float r = fmaf(lost, 1.44269504088896341f, fmaf(d, 0x1.4ae0c0p-26f, fmaf(d, 1.44269504088896341f, -t)));   // (log2 e in two parts)
    const float e = __builtin_amdgcn_exp2f(t);
    return fmaf(e, r * 0.693147180559945309f, e);
}
// Likewise, within 4 steps: the exponential of a negative argument, whatever the sign of x
__device__ __forceinline__ float sigmoid(float x) {
    const float e = exp_over(-fabsf(x), 0.0f);
    return (x < 0.0f ? e : 1.0f) * rcp_fast(1.0f + e);
}
// e^x in binary64: x = n ln 2 + r with |r| <= ln 2 / 2, the Taylor polynomial of degree 13 in r (its first missing term is
// below 2^-57), scaled by 2^n.  Within two steps of its value; arguments beyond +-800 give infinity and 0.
__device__ __forceinline__ double exp64(double x) {
    x = fmin(fmax(x, -800.0), 800.0);
    const double n = rint(x * 1.44269504088896340736);
    // ln 2 in two parts: cut behind its 41st binary place, so that 11 bits of n times it are exact, and the rest rounded to binary64
    double r = fma(n, -0x1.62e42fefa3p-1, x);
    r = fma(n, -0x1.3de6af278ece6p-42, r);
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
    const float t = rcp_fast(1.0f + exp_fast(-fabsf(x)));   // (an error of 3 |x| half steps enters with e^-|x|: 1.2 of them at most)
    return x < 0.0f ? exp_over(x, c) * t : t;
}

struct WinnersArgs {
    sdrb_winners_spec w;
    uint64_t n_rows, ld;
    uint32_t n_ids;
    uint32_t group_size, group_lanes_log2;   // ids of a group; lanes that look at one group together
    uint32_t group_magic;                    // id * group_magic >> 31 is the id's group
    uint32_t lds_groups;                     // where a row's LDS holds its groups, behind its winners and keys
    uint32_t lds_row;                        // bytes of dynamic LDS a row has
};

constexpr int kHeld = 2;   // candidates a thread takes at most
// The k for which the threads' largest keys, two a thread, give a threshold that leaves few enough candidates: half of them at most.
template <int THREADS>
constexpr uint32_t kMostByThreshold = THREADS;

// A row of scores and the steps that choose its winners.  SHARES: keys are shares (+ bias), exactly so in binary64; else the
// scores.
template <int R, int THREADS, bool SHARES, typename T>
struct Row {
    using L = Layout<R, THREADS>;
    using K = std::conditional_t<SHARES, double, float>;
    using U = std::conditional_t<SHARES, uint64_t, uint32_t>;
    static constexpr int C = L::C, Q = R / C;
    static constexpr int kDrop = SHARES ? 0 : kAlike<T>;

    const WinnersArgs& a;
    const T* s_row;
    unsigned char* mine;    // LDS of the row
    Team<THREADS> team;
    float top, inv_sum;     // of a softmax over the row
    double exact_inv_sum;   // where it enters keys

    __device__ __forceinline__ bool sig() const { return a.w.score == SDRB_SCORE_SIGMOID; }
    __device__ __forceinline__ static uint32_t thread() { return Team<THREADS>::thread(); }
    // the winners in LDS, ascending
    __device__ __forceinline__ int32_t* win_ids() const { return reinterpret_cast<int32_t*>(mine); }
    __device__ __forceinline__ float* win_scores() const { return reinterpret_cast<float*>(mine) + a.w.k; }

    __device__ __forceinline__ double exact_key(float x, uint32_t id) const {
        double key = sig() ? sigmoid((double)x) : exp64(below((double)x, (double)top)) * exact_inv_sum;
        if (a.w.bias) key += (double)a.w.bias[id];
        return x > -INFINITY && key > -INFINITY ? key + 0.0 : -INFINITY;   // (a NaN of the bias is no key; -0 is 0)
    }

    // Which of a thread's keys lie in the best groups, a bit a register.  slack: how far a key may be off, beside its own
    // rounding; where that does not tell the groups apart, they are scored by exact keys.
    __device__ __forceinline__ uint32_t in_best_groups(const float (&key)[R], float slack) {
        bool sure;
        if constexpr (C == 8) {
            const uint32_t span = a.group_size / 8;
            if (a.group_size % 8 == 0 && (span & (span - 1)) == 0 && span <= (uint32_t)Team<THREADS>::kLanes) {
                const uint32_t kept = in_best_groups_by_lanes(key, slack, span, sure);
                if (sure) return kept;
                find_best_groups<K>([&](uint32_t id) { return exact_key_of(id); }, (K)0, sure);
                return kept_of_best_ones();
            }
        }
        float* keys = reinterpret_cast<float*>(mine);
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (L::id(r) < a.n_ids) keys[L::id(r)] = key[r];
        team.sync();
        find_best_groups<float>([&](uint32_t id) { return keys[id]; }, slack, sure);
        if (!sure) find_best_groups<K>([&](uint32_t id) { return exact_key_of(id); }, (K)0, sure);
        return kept_of_best_ones();
    }
    // size: the largest sum of sizes of summed keys; worst and lost: the lowest score that is kept and the highest that is not
    template <typename F>
    __device__ __forceinline__ bool told_apart(F size, F worst, F lost, F slack) {
        size = team.max(size);
        worst = -team.max(-worst);
        lost = team.max(lost);
        // two sums, of two keys each: every one off by slack, and by three roundings of half a step of at most `size`
        return !(lost > (F)-INFINITY) || worst - lost > 4 * slack + size * (F)0x1p-21;
    }
    // Groups of 8 * span ids, span a power of two up to the lanes of the team: each lies in one chunk, with whole registers of
    // `span` neighbouring lanes.
    __device__ __forceinline__ uint32_t in_best_groups_by_lanes(const float (&key)[R], float slack, uint32_t span, bool& sure) {
        using F = float;
        const sdrb_winners_spec& w = a.w;
        const uint32_t per_chunk = THREADS / span, own = thread() / span;
        F* group = reinterpret_cast<F*>(mine);   // [groups, rounded up to 4]
        F score[Q], size = 0;
        uint32_t before[Q];
        for (uint32_t g = w.groups + thread(); g < (w.groups + 3) / 4 * 4; g += THREADS) group[g] = (F)-INFINITY;
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            F best = key[q * C], next = (F)-INFINITY;
            const auto meet = [&](F b, F n) {
                next = fmax(fmin(best, b), fmax(next, n));
                best = fmax(best, b);
            };
#pragma unroll
            for (int j = 1; j < C; ++j) {
                next = fmax(next, fmin(best, key[q * C + j]));
                best = fmax(best, key[q * C + j]);
            }
            if (span >= 2) meet(dpp<0xB1, 0xF>(best, best), dpp<0xB1, 0xF>(next, next));
            if (span >= 4) meet(dpp<0x4E, 0xF>(best, best), dpp<0x4E, 0xF>(next, next));
            if (span >= 8) meet(dpp<0x141, 0xF>(best, best), dpp<0x141, 0xF>(next, next));
            if (span >= 16) meet(dpp<0x140, 0xF>(best, best), dpp<0x140, 0xF>(next, next));
            if constexpr (THREADS >= 64) {
                if (span >= 32) meet(__shfl_xor(best, 16, 64), __shfl_xor(next, 16, 64));
                if (span >= 64) meet(__shfl_xor(best, 32, 64), __shfl_xor(next, 32, 64));
            }
            const bool two = w.group_top > 1 && next > (F)-INFINITY;
            score[q] = two ? best + next : best;
            if (best > (F)-INFINITY) size = fmax(size, fabs(best) + (two ? fabs(next) : (F)0));
            const uint32_t g = q * per_chunk + own;
            if ((thread() & (span - 1)) == 0 && g < w.groups) group[g] = score[q];
            before[q] = 0;
        }
        team.sync();
        for (uint32_t o = 0; o < w.groups; o += 4) {
            F other[4];
            __builtin_memcpy(other, group + o, sizeof other);
#pragma unroll
            for (int q = 0; q < Q; ++q)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    before[q] += other[j] > score[q] || (other[j] == score[q] && o + j < q * per_chunk + own) ? 1u : 0u;
        }
        F worst = (F)INFINITY, lost = (F)-INFINITY;
        uint32_t kept = 0;
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            const bool in = score[q] > (F)-INFINITY && before[q] < w.top_groups;
            if (in) worst = fmin(worst, score[q]);
            else lost = fmax(lost, score[q]);
            kept |= in ? 0xFFu << (q * C) : 0u;
        }
        team.sync();
        sure = !(slack > (F)0) || told_apart(size, worst, lost, slack);
        return kept;
    }
    // Any groups: 2^group_lanes_log2 threads look through a group; key_of(id) is called in a rolled loop.  A byte a group is left
    // in LDS: best_ones().
    __device__ __forceinline__ unsigned char* best_ones() const { return mine + a.lds_groups; }
    template <typename F, typename G>
    __device__ __forceinline__ void find_best_groups(G key_of, F slack, bool& sure) {
        const sdrb_winners_spec& w = a.w;
        F* group = reinterpret_cast<F*>(best_ones() + kWinnersMaxGroups);   // [groups]
        const uint32_t lanes = 1u << a.group_lanes_log2;
        F size = 0;
        for (uint32_t g0 = 0; g0 < w.groups; g0 += THREADS >> a.group_lanes_log2) {
            const uint32_t g = g0 + (thread() >> a.group_lanes_log2);
            F best = (F)-INFINITY, next = (F)-INFINITY;
            if (g < w.groups)
#pragma unroll 1
                for (uint32_t e = thread() & (lanes - 1); e < a.group_size; e += lanes) {
                    const F k = key_of(g * a.group_size + e);
                    next = fmax(next, fmin(best, k));
                    best = fmax(best, k);
                }
#pragma unroll 1
            for (uint32_t d = 1; d < lanes; d <<= 1) {
                const F b = __shfl_xor(best, (int)d, 64), n = __shfl_xor(next, (int)d, 64);
                next = fmax(fmin(best, b), fmax(next, n));
                best = fmax(best, b);
            }
            const bool two = w.group_top > 1 && next > (F)-INFINITY;
            if (g < w.groups && (thread() & (lanes - 1)) == 0) group[g] = two ? best + next : best;
            if (best > (F)-INFINITY) size = fmax(size, fabs(best) + (two ? fabs(next) : (F)0));
        }
        team.sync();
        // a group is one of the best if fewer than top_groups stand before it
        F worst = (F)INFINITY, lost = (F)-INFINITY;
#pragma unroll 1
        for (uint32_t g = thread(); g < w.groups; g += THREADS) {
            const F score = group[g];
            uint32_t before = 0;
#pragma unroll 1
            for (uint32_t o = 0; o < w.groups; ++o) before += group[o] > score || (group[o] == score && o < g) ? 1u : 0u;
            const bool in = score > (F)-INFINITY && before < w.top_groups;
            best_ones()[g] = in ? 1 : 0;
            if (in) worst = fmin(worst, score);
            else lost = fmax(lost, score);
        }
        sure = !(slack > (F)0) || told_apart(size, worst, lost, slack);
        team.sync();
    }
    __device__ __forceinline__ uint32_t kept_of_best_ones() const {
        uint32_t kept = 0;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const uint32_t g = __umulhi(2 * L::id(r), a.group_magic);
            if (L::id(r) < a.n_ids && best_ones()[g]) kept |= 1u << r;
        }
        return kept;
    }
    __device__ __forceinline__ float score_of(uint32_t id) const { return fmaxf(to_f32(s_row[id]) + 0.0f, -INFINITY); }
    __device__ __forceinline__ K exact_key_of(uint32_t id) const {
        if constexpr (SHARES) return exact_key(score_of(id), id);
        else return score_of(id);
    }

    // the winners among keys that the threads hold CH at a time, to LDS
    template <int H, int CH, typename F, typename G>
    __device__ __forceinline__ uint32_t put_winners(const U (&key)[H], F id_of, G score_of) {
        uint32_t won, here[H / CH], place[H / CH];
        const U none = order_of((K)-INFINITY) >> kDrop;
        uint32_t found;
        if constexpr (H == 1 && THREADS == 16) {
            won = key[0] > none && ranked_before<15>(key[0], thread()) < a.w.k ? 1u : 0u;
            found = team.count(won != 0);
        } else {
            found = select_largest<H, CH, THREADS>(key, none, a.w.k, team, won);
        }
#pragma unroll
        for (int q = 0; q < H / CH; ++q) here[q] = __popc((won >> (q * CH)) & (uint32_t)((1ull << CH) - 1));
        team.places(here, place);
#pragma unroll
        for (int j = 0; j < H; ++j)
            if ((won >> j) & 1u) {
                win_ids()[place[j / CH]] = id_of(j);
                win_scores()[place[j / CH]++] = score_of(j);
            }
        team.sync();
        return found;
    }

    // whether the ids of these registers have the same score and bias, in all threads
    __device__ __forceinline__ bool alike(uint32_t bits) {
        uint32_t least[2] = {0xFFFFFFFFu, 0xFFFFFFFFu}, most[2] = {0u, 0u};
#pragma unroll 1
        while (bits) {
            const uint32_t id = L::id(__builtin_ctz(bits));
            const uint32_t of[2] = {order_of(score_of(id)), a.w.bias ? order_of(a.w.bias[id] + 0.0f) : 0u};
            bits &= bits - 1;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                least[i] = of[i] < least[i] ? of[i] : least[i];
                most[i] = max_u32(most[i], of[i]);
            }
        }
        const bool scores = team.min(least[0]) == team.max(most[0]);
        const bool biases = !a.w.bias || team.min(least[1]) == team.max(most[1]);
        return scores && biases;
    }
    // the candidates that a threshold leaves, and the winners among them; false where the row needs choose_among_all
    __device__ __forceinline__ bool choose_among_candidates(float (&key)[R], uint32_t& found) {
        const sdrb_winners_spec& w = a.w;
        float slack = 0.0f;
        if constexpr (SHARES) {
            // Off by less than 3.1 * 2^-24 for the sigmoid -- 1.5 |x| + 2 steps in its exponential t, which enter the result
            // with t / (1 + t)^2, and two roundings.  A softmax's share e^-d / sum is off by 3 d + 4 times 2^-24 of itself -- d, its
            // product with log2 e and that constant, a step of the exponential, and two roundings -- and so by less than
            // 4.1 * 2^-24 of the largest share there can be, 1 / sum: (3 d + 4) e^-d falls from 4 on.
            slack = sig() ? 0x1p-22f : inv_sum * 0x1p-21f;
            float b[R];
            if (w.bias) read_row<R, THREADS>(w.bias, a.n_ids, 0.0f, b);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float k = sig() ? sigmoid_fast(key[r]) : exp_fast(below(key[r], top)) * inv_sum;
                if (w.bias) k = fmaxf(k + b[r], -INFINITY);
                key[r] = key[r] > -INFINITY ? k : -INFINITY;
            }
        }
        if (w.groups > 1) {
            const uint32_t kept = in_best_groups(key, slack);
#pragma unroll
            for (int r = 0; r < R; ++r) key[r] = (kept >> r) & 1u ? key[r] : -INFINITY;
            team.sync();
        }

        constexpr int kTops = R > 1 ? 2 : 1;
        uint32_t tops[kTops];
#pragma unroll
        for (int h = 0; h < kTops; ++h) {
            float most = key[h * (R / kTops)];
#pragma unroll
            for (int r = 1; r < R / kTops; ++r) most = fmaxf(most, key[h * (R / kTops) + r]);
            tops[h] = order_of(most) >> kDrop;
        }
        constexpr uint32_t none = kOrderOfNone >> kDrop;
        // the key from which on `count` finds k keys, or close to it: at least k are >= lo
        const auto find = [&](uint32_t& lo, uint32_t hi, auto count) {
            uint32_t c = 0;
#pragma unroll 1
            while (hi - lo > 1 && c != w.k) {
                const uint32_t mid = lo + (hi - lo) / 2;
                c = count(mid);
                if (c >= w.k) lo = mid;
                else hi = mid;
            }
        };
        uint32_t bits = 0;
        uint32_t here[Q], place[Q], n, lo = none, most = 0;
        const auto placed = [&]() {
#pragma unroll
            for (int q = 0; q < Q; ++q) here[q] = __popc((bits >> (q * C)) & ((1u << C) - 1u));
            return team.places(here, place);
        };
        const auto collect = [&](float t) {
            bits = 0;
#pragma unroll
            for (int r = 0; r < R; ++r) bits |= key[r] >= t ? 1u << r : 0u;
            return placed();
        };
        // Where k approximate keys are no smaller than t, and fewer are larger, the winners are no smaller than t - off: the k-th
        // may seem larger than it is, and another one smaller.  (Every key > -inf.  A bias makes a key infinite, not its rounding: an
        // infinite t is off by nothing.)
        const auto off = [&](float t) { return SHARES && t < INFINITY ? 2.0f * slack + fabsf(t) * 0x1p-21f : 0.0f; };
        const auto lowered = [&](float t) { return fmaxf(SHARES ? t - off(t) : t, -3.402823466e38f); };
        if (w.k <= kMostByThreshold<THREADS> && team.template count_all<kTops>([&](int h) { return tops[h] > none; }) >= w.k) {
            uint32_t least = 0xFFFFFFFFu;
#pragma unroll
            for (int h = 0; h < kTops; ++h) least = tops[h] > none && tops[h] < least ? tops[h] : least;
            lo = team.min(least);
        }
#pragma unroll
        for (int h = 0; h < kTops; ++h) most = max_u32(most, tops[h]);
        most = team.max(most) + 1;
        if (lo > none) find(lo, most, [&](uint32_t mid) { return team.template count_all<kTops>([&](int h) { return tops[h] >= mid; }); });
        n = collect(lowered(key_at(lo << kDrop)));
        if (n > (uint32_t)THREADS * kHeld) {
            // too many: k of all keys instead of k of the largest
            if (lo == none) lo = none + 1;
            find(lo, most, [&](uint32_t mid) {
                const float t = key_at(mid << kDrop);
                return team.template count_all<R>([&](int r) { return key[r] >= t; });
            });
            const float t = key_at(lo << kDrop);
            // keys that are larger for sure -- none where the k-th is infinite -- and those that may be the k-th
            const float larger = !(t < INFINITY) ? NAN : SHARES ? t + off(t) : key_at((lo + 1) << kDrop);
            const uint32_t more = w.k - collect(larger);
            const uint32_t sure = bits;
            n = collect(lowered(t));
            if (n > (uint32_t)THREADS * kHeld) {
                // too many may be the k-th: where they are equal, the lowest ids fill the places
                bits &= ~sure;
                if (SHARES && more && t < INFINITY && !alike(bits)) return false;
                placed();
                uint32_t taken = sure;
#pragma unroll
                for (int r = 0; r < R; ++r)
                    if ((bits >> r) & 1u) taken |= place[r / C]++ < more ? 1u << r : 0u;
                bits = taken;
                n = placed();
            }
        }
        int32_t* list = reinterpret_cast<int32_t*>(mine);
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            uint32_t b = (bits >> (q * C)) & ((1u << C) - 1u), at = place[q];
            while (b) {
                list[at++] = (int32_t)(L::id(q * C) + (uint32_t)__builtin_ctz(b));
                b &= b - 1;
            }
        }
        team.sync();
        found = n <= THREADS ? choose_from_list<1>(list, n) : choose_from_list<kHeld>(list, n);
        return true;
    }
    template <int H>
    __device__ __forceinline__ uint32_t choose_from_list(const int32_t* list, uint32_t n) {
        U key[H];
        float x[H];
        int32_t id[H];
#pragma unroll
        for (int j = 0; j < H; ++j) {
            const uint32_t i = j * THREADS + thread();
            key[j] = 0;
            x[j] = -INFINITY;
            id[j] = -1;
            if (i < n) {
                id[j] = list[i];
                x[j] = to_f32(s_row[id[j]]) + 0.0f;   // -0 is 0
                if constexpr (SHARES) key[j] = order_of(exact_key(x[j], (uint32_t)id[j]));
                else key[j] = order_of(x[j]) >> kDrop;
            }
        }
        team.sync();   // the list has been read: winners are put in its place
        return put_winners<H, 1>(key, [&](int j) { return id[j]; }, [&](int j) { return x[j]; });
    }

    // bisection over all keys, computed anew in every step
    __device__ __forceinline__ uint32_t choose_among_all() {
        const sdrb_winners_spec& w = a.w;
        bool sure;
        if (w.groups > 1) find_best_groups<K>([&](uint32_t id) { return exact_key_of(id); }, (K)0, sure);
        const U none = order_of((K)-INFINITY);
        const auto order_at = [&](uint32_t id) {
            if (w.groups > 1 && !best_ones()[__umulhi(2 * id, a.group_magic)]) return (U)0;
            return order_of(exact_key_of(id));
        };
        const auto count = [&](U least) {
            uint32_t c = 0;
#pragma unroll 1
            for (uint32_t id = thread(); id < a.n_ids; id += THREADS) c += order_at(id) >= least ? 1u : 0u;
            return team.sum(c);
        };
        // at least min(k, live) keys are >= lo, fewer than k >= hi
        U lo = none + 1, hi = ~(U)0;
        uint32_t above = 0;   // keys above lo where the bisection ends on a key
        uint32_t c = count(lo);
        if (c > w.k) {
#pragma unroll 1
            while (hi - lo > 1 && c != w.k) {
                const U mid = lo + (hi - lo) / 2;
                c = count(mid);
                if (c >= w.k) lo = mid;
                else hi = mid;
            }
            if (c != w.k) above = count(lo + 1);
        }
        uint32_t room = w.k - above, found = 0;   // places for keys equal to lo
        const bool ties = above != 0 || c > w.k || hi - lo <= 1;
#pragma unroll 1
        for (uint32_t id0 = 0; id0 < a.n_ids; id0 += THREADS) {
            const uint32_t id = id0 + thread();
            const U key = id < a.n_ids ? order_at(id) : (U)0;
            bool win = key >= lo;
            uint32_t here[1], place[1];
            if (ties) {
                here[0] = key == lo ? 1u : 0u;
                const uint32_t equal = team.places(here, place);
                if (here[0] && place[0] >= room) win = false;
                room -= equal < room ? equal : room;
            }
            here[0] = win ? 1u : 0u;
            const uint32_t wins = team.places(here, place);
            if (win) {
                win_ids()[found + place[0]] = (int32_t)id;
                win_scores()[found + place[0]] = score_of(id);
            }
            found += wins;
        }
        team.sync();
        return found;
    }
};

constexpr uint32_t block_of(int threads) { return threads <= 64 ? 256 : threads; }

template <int R, int THREADS, bool SHARES, typename T>
__global__ __launch_bounds__(block_of(THREADS)) void k_winners(WinnersArgs a, const T* __restrict__ scores, int32_t* __restrict__ out_ids,
                                                               float* __restrict__ out_weights) {
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    constexpr int kWaves = THREADS > 64 ? THREADS / 64 : 1;
    __shared__ double slots[2 * kWaves];
    __shared__ uint32_t starts[kWaves > 1 ? 8 * kWaves : 1];
    const uint32_t in_block = threadIdx.x / THREADS;
    const uint64_t row = (uint64_t)blockIdx.x * (block_of(THREADS) / THREADS) + in_block;
    if (row >= a.n_rows) return;
    const sdrb_winners_spec& w = a.w;
    Row<R, THREADS, SHARES, T> x{a, scores + row * a.ld, lds + in_block * a.lds_row, {slots, starts, 0}, 0.0f, 0.0f, 0.0};
    const bool sig = x.sig();
    uint32_t found = 0;
    [[maybe_unused]] bool chosen;
    {
        float s[R];
        read_scores<R, THREADS>(x.s_row, a.n_ids, s);
        if (!sig && (SHARES || !w.renormalise)) {   // a softmax over the row
            float m = s[0];
#pragma unroll
            for (int r = 1; r < R; ++r) m = fmaxf(m, s[r]);
            x.top = x.team.max(m);
            if constexpr (SHARES) {
                double sum = 0.0;
#pragma unroll
                for (int r = 0; r < R; ++r)
                    if (s[r] > -INFINITY) sum += exp64(below((double)s[r], (double)x.top));
                x.exact_inv_sum = 1.0 / x.team.sum(sum);
                x.inv_sum = (float)x.exact_inv_sum;
            } else {
                float sum = 0.0f;
#pragma unroll
                for (int r = 0; r < R; ++r)
                    if (s[r] > -INFINITY) sum += exp_fast(below(s[r], x.top));
                x.inv_sum = rcp_fast(x.team.sum(sum));
            }
        }
        chosen = x.choose_among_candidates(s, found);
    }
    if constexpr (SHARES) {
        if (!chosen) {
            x.team.sync();
            found = x.choose_among_all();
        }
    }

    // the weights, a winner a thread
    const uint32_t thread = x.thread();
    const int32_t* win_id = x.win_ids();
    const float* win_s = x.win_scores();
    float shift = 0.0f, norm = w.scale;
    if (w.renormalise) {
        float m = -INFINITY;
        for (uint32_t i = thread; i < found; i += THREADS) m = max_of(m, win_s[i]);
        shift = x.team.max(m);
        if (sig) shift = shift < 0.0f ? shift : 0.0f;
        float sum = 0.0f;
        for (uint32_t i = thread; i < found; i += THREADS) sum += sig ? sigmoid_over(win_s[i], shift) : exp_over(win_s[i], shift);
        norm = w.scale * rcp_fast(x.team.sum(sum));
    }
    int32_t* ids = out_ids + row * w.k;
    float* weights = out_weights + row * w.k;
    for (uint32_t i = thread; i < w.k; i += THREADS) {
        int32_t id = -1;
        float weight = 0.0f;
        if (i < found) {
            id = win_id[i];
            const float v = win_s[i];
            if (sig) weight = norm * (w.renormalise ? sigmoid_over(v, shift) : sigmoid(v));
            else weight = norm * (w.renormalise ? exp_over(v, shift) : exp_over(v, x.top) * x.inv_sum);
        }
        ids[i] = id;
        weights[i] = weight;
    }
}

struct WinnersGradArgs {
    sdrb_winners_spec w;
    uint64_t n_rows, ld, out_ld;
    uint32_t n_ids;
};

// d scores of a row, from its winners and their weights' gradient.  The row is written as if nothing had won -- zeros, or a
// softmax's share of what is taken from every score -- and the winners' values are stored over it, once those stores have
// arrived; only a softmax over the whole row reads it, the other gradients read the winners' scores alone.  No LDS: what
// bounds it is latency (ids, then their scores) over the waves in flight, and the write of the result.
template <int R, int THREADS, bool WHOLE, typename T, typename O>
__global__ __launch_bounds__(block_of(THREADS)) void k_winners_grad(WinnersGradArgs a, const T* __restrict__ scores,
                                                                    const int32_t* __restrict__ ids_in,
                                                                    const float* __restrict__ grad_in, O* out) {
    using L = Layout<R, THREADS>;
    constexpr int C = L::C, kWaves = THREADS > 64 ? THREADS / 64 : 1;
    __shared__ double slots[2 * kWaves];
    const uint64_t row = (uint64_t)blockIdx.x * (block_of(THREADS) / THREADS) + threadIdx.x / THREADS;
    if (row >= a.n_rows) return;
    Team<THREADS> team{slots, nullptr, 0};
    const uint32_t thread = team.thread();
    const T* s_row = scores + row * a.ld;
    O* to = out + row * a.out_ld;
    const sdrb_winners_spec& w = a.w;
    const bool sig = w.score == SDRB_SCORE_SIGMOID;
    // a thread's winners (the layouts give it at most two); -1 where it has none: a NaN or -inf never won
    constexpr int H = 2;
    int32_t id[H];
    float x[H], g[H];
#pragma unroll
    for (int h = 0; h < H; ++h) {
        const uint32_t i = h * THREADS + thread;
        id[h] = i < w.k ? ids_in[row * w.k + i] : -1;
        g[h] = i < w.k ? grad_in[row * w.k + i] : 0.0f;
    }
    float s[WHOLE ? R : 1];
    if constexpr (WHOLE) {
        read_scores<R, THREADS>(s_row, a.n_ids, s);
    } else {
        constexpr int V = 16 / sizeof(O);
        const float zeros[V] = {};
        for (uint32_t first = thread * V; first < a.n_ids; first += THREADS * V) {
            if (first + V <= a.n_ids) {
                store_n<V>(to + first, zeros);
            } else {
                for (uint32_t j = first; j < a.n_ids; ++j) to[j] = from_f32<O>(0.0f);
            }
        }
    }
#pragma unroll
    for (int h = 0; h < H; ++h) {
        x[h] = id[h] >= 0 && (uint32_t)id[h] < a.n_ids ? to_f32(s_row[id[h]]) : -INFINITY;
        if (!(x[h] > -INFINITY)) id[h] = -1;
    }
    // the part of the softmax that the sum runs over; `shift` is its largest argument
    float shift = 0.0f, inv = 1.0f, dot = 0.0f;
    const auto part_of = [&](float v) { return sig ? sigmoid_over(v, shift) : exp_over(v, shift); };
    if (WHOLE || w.renormalise) {
        float m = -INFINITY, sum = 0.0f;
        if constexpr (WHOLE) {
#pragma unroll
            for (int r = 0; r < R; ++r) m = fmaxf(m, s[r]);
        } else {
#pragma unroll
            for (int h = 0; h < H; ++h)
                if (id[h] >= 0) m = fmaxf(m, x[h]);
        }
        shift = team.max(m);
        if (sig) shift = shift < 0.0f ? shift : 0.0f;
        if constexpr (WHOLE) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                // (a share d below the largest by 3 d half steps of its own, so by 1.2 half steps of the largest at most; with exp_over
                // 8192 rows of 2048 bf16 scores took 19.3 us, not 16.0)
                s[r] = s[r] > -INFINITY ? exp_fast(below(s[r], shift)) : 0.0f;
                sum += s[r];
            }
        }
#pragma unroll
        for (int h = 0; h < H; ++h)
            if (id[h] >= 0) {
                const float p = part_of(x[h]);
                if (!WHOLE) sum += p;
                dot = fmaf(p, g[h], dot);
            }
        inv = rcp_fast(team.sum(sum));
        dot = team.sum(dot) * inv;
    }
    if constexpr (WHOLE) {
        const float scale = -w.scale * inv * dot;
#pragma unroll
        for (int q = 0; q < R / C; ++q) {
            const uint32_t first = L::id(q * C);
            float part[C];
#pragma unroll
            for (int j = 0; j < C; ++j) part[j] = s[q * C + j] > 0.0f ? scale * s[q * C + j] : 0.0f;   // (a row without live scores has inv = inf)
            if (first + C <= a.n_ids) {
                store_n<C>(to + first, part);
            } else {
#pragma unroll
                for (int j = 0; j < C; ++j)
                    if (first + j < a.n_ids) to[first + j] = from_f32<O>(part[j]);
            }
        }
    }
    // the stores above come from other lanes: they have arrived before the ones below set out
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0)
    if constexpr (kWaves > 1) __syncthreads();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int h = 0; h < H; ++h)
        if (id[h] >= 0) {
            float d = WHOLE || w.renormalise ? part_of(x[h]) * inv * (g[h] - dot) : g[h] * sigmoid(x[h]);
            if (sig) d *= sigmoid(-x[h]);
            to[id[h]] = from_f32<O>(w.scale * d);
        }
}

// Calls f(R, THREADS) for rows of n ids, k of which win: as few waves as hold the ids in 32 registers and choose k of them by a
// threshold.  Waves that meet in LDS at every step of a bisection cost more than registers do: 4096 rows of 4096 ids, k = 40,
// take 22.6 us with two waves a row and 72.7 with eight, 64 such rows 8.9 and 13.5, a single one 8.5 and 13.0.  (Beyond 32 the
// registers cost more: 4096 rows of 16384 ids, k = 328, 122 us with eight waves and 191 with four.)
// Four rows share a wave where rows are short and enough of them to fill the chip that way (1024 SIMDs, a wave each); with fewer
// the row's latency counts, and 64 lanes have less to do each.
template <typename F>
int with_layout(uint32_t n, uint64_t n_rows, uint32_t k, F&& f) {
    using std::integral_constant;
    const auto lanes = integral_constant<int, 16>{};
    const auto wave = integral_constant<int, 64>{};
    const auto two = integral_constant<int, 128>{};
    const auto four = integral_constant<int, 256>{};
    const auto eight = integral_constant<int, 512>{};
    if (n <= 256 && n_rows >= 4096 && k <= kMostByThreshold<16>) {
        if (n <= 64) return f(integral_constant<int, 4>{}, lanes);
        if (n <= 128) return f(integral_constant<int, 8>{}, lanes);
        return f(integral_constant<int, 16>{}, lanes);
    }
    if (n <= 64) return f(integral_constant<int, 1>{}, wave);
    if (n <= 128) return f(integral_constant<int, 2>{}, wave);
    if (n <= 2048 && k <= kMostByThreshold<64>) {
        if (n <= 256) return f(integral_constant<int, 4>{}, wave);
        if (n <= 512) return f(integral_constant<int, 8>{}, wave);
        if (n <= 1024) return f(integral_constant<int, 16>{}, wave);
        return f(integral_constant<int, 32>{}, wave);
    }
    if (n <= 4096 && k <= kMostByThreshold<128>) {
        if (n <= 1024) return f(integral_constant<int, 8>{}, two);
        if (n <= 2048) return f(integral_constant<int, 16>{}, two);
        return f(integral_constant<int, 32>{}, two);
    }
    if (n <= 8192 && k <= kMostByThreshold<256>) {
        if (n <= 2048) return f(integral_constant<int, 8>{}, four);
        if (n <= 4096) return f(integral_constant<int, 16>{}, four);
        return f(integral_constant<int, 32>{}, four);
    }
    if (n <= 1024) return f(integral_constant<int, 2>{}, eight);
    if (n <= 4096) return f(integral_constant<int, 8>{}, eight);
    if (n <= 8192) return f(integral_constant<int, 16>{}, eight);
    return f(integral_constant<int, 32>{}, eight);
}
// The same for the gradient, where k counts only because a thread takes two winners at most.  (Without a softmax over the whole row
// nothing is held in registers.)
template <typename F>
int with_grad_layout(bool whole, uint32_t n, uint64_t n_rows, uint32_t k, F&& f) {
    using std::integral_constant;
    const auto go = [&](auto r, auto threads) { return whole ? f(r, threads, std::true_type{}) : f(integral_constant<int, 1>{}, threads, std::false_type{}); };
    const auto lanes = integral_constant<int, 16>{};
    const auto wave = integral_constant<int, 64>{};
    if (n <= 256 && n_rows >= 4096 && k <= 32) {
        if (n <= 64) return go(integral_constant<int, 4>{}, lanes);
        if (n <= 128) return go(integral_constant<int, 8>{}, lanes);
        return go(integral_constant<int, 16>{}, lanes);
    }
    if (n <= 2048 && k <= 128) {
        if (n <= 64) return go(integral_constant<int, 1>{}, wave);
        if (n <= 256) return go(integral_constant<int, 4>{}, wave);
        if (n <= 512) return go(integral_constant<int, 8>{}, wave);
        if (n <= 1024) return go(integral_constant<int, 16>{}, wave);
        return go(integral_constant<int, 32>{}, wave);
    }
    if (n <= 4096 && k <= 256) return go(integral_constant<int, 32>{}, integral_constant<int, 128>{});
    if (n <= 8192 && k <= 512) return go(integral_constant<int, 32>{}, integral_constant<int, 256>{});
    return go(integral_constant<int, 32>{}, integral_constant<int, 512>{});
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
    return with_layout(a.n_ids, a.n_rows, spec.k, [&](auto r, auto n_threads) {
        constexpr int R = decltype(r)::value, THREADS = decltype(n_threads)::value;
        constexpr uint32_t kPerBlock = block_of(THREADS) / THREADS;
        a.group_lanes_log2 = 0;
        while (a.group_lanes_log2 < 6 && (spec.groups << (a.group_lanes_log2 + 1)) <= (uint32_t)THREADS) ++a.group_lanes_log2;
        return with_type(scores.type, [&](auto t) {
            using T = decltype(t);
            const auto go = [&](auto s) {
                constexpr bool SHARES = decltype(s)::value;
                const auto up = [](size_t bytes) { return (uint32_t)((bytes + 15) / 16 * 16); };
                const size_t held = (a.n_ids < (uint32_t)THREADS * kHeld ? a.n_ids : (uint32_t)THREADS * kHeld) * sizeof(int32_t);
                const size_t keys = spec.groups > 1 ? a.n_ids * sizeof(float) : 0, won = spec.k * 8;
                a.lds_groups = up(won > held ? (won > keys ? won : keys) : (held > keys ? held : keys));
                a.lds_row = a.lds_groups + (spec.groups > 1 ? up(kWinnersMaxGroups + (spec.groups + 3) * (SHARES ? sizeof(double) : sizeof(float))) : 0);
                const size_t lds = (size_t)a.lds_row * kPerBlock;
                if (const int rc = allow_lds(&k_winners<R, THREADS, SHARES, T>, lds)) return rc;
                return in_launches((scores.n_rows + kPerBlock - 1) / kPerBlock, block_of(THREADS), [&](uint64_t first, uint32_t blocks) {
                    const uint64_t row = first * kPerBlock;
                    a.n_rows = scores.n_rows - row;
                    hipLaunchKernelGGL((k_winners<R, THREADS, SHARES, T>), dim3(blocks), dim3(block_of(THREADS)), lds, stream, a,
                                       static_cast<const T*>(scores.data) + row * a.ld, ids + row * spec.k, weights + row * spec.k);
                    SDRB_HIP(hipGetLastError());
                    return SDRB_OK;
                });
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
    return with_grad_layout(spec.score == SDRB_SCORE_SOFTMAX && !spec.renormalise, a.n_ids, a.n_rows, spec.k, [&](auto r, auto n_threads, auto all) {
        constexpr int R = decltype(r)::value, THREADS = decltype(n_threads)::value;
        constexpr bool WHOLE = decltype(all)::value;
        constexpr uint32_t kPerBlock = block_of(THREADS) / THREADS;
        return with_type(scores.type, [&](auto t) {
            return with_type(out.type, [&](auto o) {
                using T = decltype(t);
                using O = decltype(o);
                return in_launches((scores.n_rows + kPerBlock - 1) / kPerBlock, block_of(THREADS), [&](uint64_t first, uint32_t blocks) {
                    const uint64_t row = first * kPerBlock;
                    a.n_rows = scores.n_rows - row;
                    hipLaunchKernelGGL((k_winners_grad<R, THREADS, WHOLE, T, O>), dim3(blocks), dim3(block_of(THREADS)), 0, stream, a,
                                       static_cast<const T*>(scores.data) + row * a.ld, ids + row * spec.k, grad_weights + row * spec.k,
                                       static_cast<O*>(out.data) + row * a.out_ld);
                    SDRB_HIP(hipGetLastError());
                    return SDRB_OK;
                });
            });
        });
    });
}

}  // namespace sdrb
