// The k winners of every row of dense scores, with their weights, and the gradient of those weights to the scores.
//
// Shares: u = softmax of a row's live scores, or their sigmoids; a score of -inf or NaN is not live.  Keys: u + bias, or the
// scores where nothing is added to the shares (the same order).  A group's score is the sum of its one or two largest
// keys; the k largest keys inside the best groups win, ties go to the lowest group and id.  Keys are compared in binary64:
// whether an id wins hangs on the difference of two of them, which binary32 exponentials would decide by their own error.
// Weights: scale * u, or, renormalised, scale * p with p = u / sum of the winners' u -- a softmax over the winners of
// l = s (softmax) or l = log sigmoid(s), which holds where every u underflows.
#include "dense_rows.h"

namespace sdrb {

namespace {

constexpr uint32_t kThreads = 256;

__device__ __forceinline__ bool live_score(float s) { return s > -INFINITY; }
__device__ __forceinline__ double sigmoid(double x) { return 1.0 / (1.0 + exp(-x)); }
// x - m for an exponential whose largest argument is m: infinities of the same sign differ by nothing
__device__ __forceinline__ double below(double x, double m) { return x == m ? 0.0 : x - m; }
__device__ __forceinline__ double logit(double x, bool sig) { return sig ? fmin(x, 0.0) - log1p(exp(-fabs(x))) : x; }

template <typename F>
__device__ __forceinline__ double block_reduce(double v, double* shared, F op) {
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1) v = op(v, __shfl_xor(v, s, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
    __syncthreads();
    v = shared[0];
    for (uint32_t k = 1; k < kThreads / 64; ++k) v = op(v, shared[k]);
    return v;
}
__device__ __forceinline__ double block_max(double v, double* shared) {
    return block_reduce(v, shared, [](double a, double b) { return a > b ? a : b; });
}
__device__ __forceinline__ double block_sum(double v, double* shared) {
    return block_reduce(v, shared, [](double a, double b) { return a + b; });
}

// the position of the largest key, the lowest of equal ones; every key must be > -inf to count
__device__ __forceinline__ int block_best(const double* key, uint32_t n, double* shared_v, int* shared_i) {
    double best = -INFINITY;
    int at = -1;
    for (uint32_t e = threadIdx.x; e < n; e += kThreads)
        if (key[e] > best) {
            best = key[e];
            at = (int)e;
        }
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1) {
        const double v = __shfl_xor(best, s, 64);
        const int i = __shfl_xor(at, s, 64);
        if (i >= 0 && (v > best || (v == best && (at < 0 || i < at)))) {
            best = v;
            at = i;
        }
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        shared_v[threadIdx.x >> 6] = best;
        shared_i[threadIdx.x >> 6] = at;
    }
    __syncthreads();
    best = shared_v[0];
    at = shared_i[0];
    for (uint32_t k = 1; k < kThreads / 64; ++k)
        if (shared_i[k] >= 0 && (shared_v[k] > best || (shared_v[k] == best && (at < 0 || shared_i[k] < at)))) {
            best = shared_v[k];
            at = shared_i[k];
        }
    __syncthreads();
    return at;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void k_winners(const T* __restrict__ scores, uint64_t ld, uint32_t n_ids, sdrb_winners_spec w,
                                                      int32_t* __restrict__ out_ids, float* __restrict__ out_weights) {
    extern __shared__ double key[];   // [n_ids], then the groups' [groups]
    __shared__ double sv[4];
    __shared__ int si[4];
    __shared__ uint32_t won[kWinnersMaxIds / 32];
    double* group = key + n_ids;
    const uint64_t row = blockIdx.x;
    const T* s = scores + row * ld;
    const bool sig = w.score == SDRB_SCORE_SIGMOID;
    const bool shares = w.bias || (w.groups > 1 && w.group_top > 1);
    double top = -INFINITY, sum = 1.0;
    if (!sig) {
        for (uint32_t e = threadIdx.x; e < n_ids; e += kThreads) top = fmax(top, (double)to_f32(s[e]));   // (a NaN is passed over)
        top = block_max(top, sv);
        sum = 0.0;
        for (uint32_t e = threadIdx.x; e < n_ids; e += kThreads)
            if (live_score(to_f32(s[e]))) sum += exp(below(to_f32(s[e]), top));
        sum = block_sum(sum, sv);
    }
    const auto share = [&](double x) { return sig ? sigmoid(x) : exp(below(x, top)) / sum; };
    for (uint32_t e = threadIdx.x; e < n_ids; e += kThreads) {
        const float x = to_f32(s[e]);
        double k = -INFINITY;
        if (live_score(x)) k = shares ? share(x) + (w.bias ? (double)w.bias[e] : 0.0) : (double)x;
        key[e] = k > -INFINITY ? k : -INFINITY;
    }
    for (uint32_t i = threadIdx.x; i < (n_ids + 31) / 32; i += kThreads) won[i] = 0;
    __syncthreads();
    if (w.groups > 1) {
        const uint32_t size = n_ids / w.groups;
        for (uint32_t g = threadIdx.x; g < w.groups; g += kThreads) {
            double a = -INFINITY, b = -INFINITY;
            for (uint32_t e = g * size; e < (g + 1) * size; ++e) {
                const double k = key[e];
                b = k > a ? a : (k > b ? k : b);
                a = k > a ? k : a;
            }
            group[g] = w.group_top > 1 && b > -INFINITY ? a + b : a;
        }
        __syncthreads();
        for (uint32_t t = 0; t < w.top_groups; ++t) {   // the best groups are marked by -inf
            const int g = block_best(group, w.groups, sv, si);
            if (g < 0) break;
            if (threadIdx.x == 0) {
                group[g] = -INFINITY;
                won[g >> 5] |= 1u << (g & 31);
            }
            __syncthreads();
        }
        for (uint32_t e = threadIdx.x; e < n_ids; e += kThreads)
            if (!(won[(e / size) >> 5] >> ((e / size) & 31) & 1u)) key[e] = -INFINITY;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < (n_ids + 31) / 32; i += kThreads) won[i] = 0;
        __syncthreads();
    }
    uint32_t found = 0;
    double best_logit = -INFINITY, logits = 0.0;
    for (; found < w.k; ++found) {
        const int e = block_best(key, n_ids, sv, si);
        if (e < 0) break;
        if (threadIdx.x == 0) {
            key[e] = -INFINITY;
            won[e >> 5] |= 1u << (e & 31);
        }
        best_logit = fmax(best_logit, logit(to_f32(s[e]), sig));
        __syncthreads();
    }
    int32_t* ids = out_ids + row * w.k;
    float* weights = out_weights + row * w.k;
    // ascending ids: a winner's place is the number of winners below it
    for (uint32_t e = threadIdx.x; e < n_ids; e += kThreads) {
        if (!(won[e >> 5] >> (e & 31) & 1u)) continue;
        uint32_t place = __popc(won[e >> 5] & ((1u << (e & 31)) - 1u));
        for (uint32_t i = 0; i < (e >> 5); ++i) place += __popc(won[i]);
        ids[place] = (int32_t)e;
        if (w.renormalise) logits += exp(below(logit(to_f32(s[e]), sig), best_logit));
        else weights[place] = (float)((double)w.scale * share(to_f32(s[e])));
    }
    if (w.renormalise) {
        logits = block_sum(logits, sv);
        for (uint32_t e = threadIdx.x; e < n_ids; e += kThreads) {
            if (!(won[e >> 5] >> (e & 31) & 1u)) continue;
            uint32_t place = __popc(won[e >> 5] & ((1u << (e & 31)) - 1u));
            for (uint32_t i = 0; i < (e >> 5); ++i) place += __popc(won[i]);
            weights[place] = (float)((double)w.scale * exp(below(logit(to_f32(s[e]), sig), best_logit)) / logits);
        }
    }
    for (uint32_t i = found + threadIdx.x; i < w.k; i += kThreads) {
        ids[i] = -1;
        weights[i] = 0.0f;
    }
}

// d scores of a row, from its winners and their weights' gradient
template <typename T, typename O>
__global__ __launch_bounds__(kThreads) void k_winners_grad(const T* __restrict__ scores, uint64_t ld, uint32_t n_ids, sdrb_winners_spec w,
                                                           const int32_t* __restrict__ ids_in, const float* __restrict__ grad_in,
                                                           O* __restrict__ out, uint64_t out_ld) {
    extern __shared__ double grad_of[];   // [n_ids]: the gradient at a winner; elsewhere 0
    __shared__ double sv[4];
    __shared__ uint32_t won[kWinnersMaxIds / 32];
    const uint64_t row = blockIdx.x;
    const T* s = scores + row * ld;
    const int32_t* ids = ids_in + row * w.k;
    const float* grad = grad_in + row * w.k;
    const bool sig = w.score == SDRB_SCORE_SIGMOID;
    for (uint32_t i = threadIdx.x; i < (n_ids + 31) / 32; i += kThreads) won[i] = 0;
    for (uint32_t e = threadIdx.x; e < n_ids; e += kThreads) grad_of[e] = 0.0;
    __syncthreads();
    const auto winner = [&](uint32_t i) { return ids[i] >= 0 && (uint32_t)ids[i] < n_ids && live_score(to_f32(s[ids[i]])); };
    for (uint32_t i = threadIdx.x; i < w.k; i += kThreads)
        if (winner(i)) {
            grad_of[ids[i]] = grad[i];
            atomicOr(&won[ids[i] >> 5], 1u << (ids[i] & 31));
        }
    __syncthreads();
    const bool whole = !sig && !w.renormalise;   // a softmax over every live score
    double top = -INFINITY, sum = 0.0, dot = 0.0;
    const auto counts = [&](uint32_t e) { return whole ? live_score(to_f32(s[e])) : (won[e >> 5] >> (e & 31) & 1u) != 0; };
    if (whole || w.renormalise) {
        for (uint32_t e = threadIdx.x; e < n_ids; e += kThreads)
            if (counts(e)) top = fmax(top, logit(to_f32(s[e]), sig));
        top = block_max(top, sv);
        for (uint32_t e = threadIdx.x; e < n_ids; e += kThreads)
            if (counts(e)) {
                const double p = exp(below(logit(to_f32(s[e]), sig), top));
                sum += p;
                dot += p * grad_of[e];
            }
        sum = block_sum(sum, sv);
        dot = block_sum(dot, sv) / sum;
    }
    for (uint32_t e = threadIdx.x; e < n_ids; e += kThreads) {
        double d = 0.0;
        if (counts(e)) {
            const double x = to_f32(s[e]);
            if (whole || w.renormalise) {
                d = exp(below(logit(x, sig), top)) / sum * (grad_of[e] - dot);
                if (sig) d *= sigmoid(-x);
            } else {
                d = grad_of[e] * sigmoid(x) * sigmoid(-x);
            }
        }
        out[row * out_ld + e] = from_f32<O>((float)((double)w.scale * d));
    }
}

}  // namespace

int launch_winners(const sdrb_dense& scores, const sdrb_winners_spec& spec, int32_t* ids, float* weights, hipStream_t stream) {
    const uint32_t n_ids = (uint32_t)scores.n_cols;
    const size_t lds = (size_t)(n_ids + spec.groups) * sizeof(double);
    return with_type(scores.type, [&](auto t) {
        using T = decltype(t);
        SDRB_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&k_winners<T>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
        hipLaunchKernelGGL((k_winners<T>), dim3((uint32_t)scores.n_rows), dim3(kThreads), lds, stream, static_cast<const T*>(scores.data),
                           scores.ld, n_ids, spec, ids, weights);
        SDRB_HIP(hipGetLastError());
        return SDRB_OK;
    });
}

int launch_winners_grad(const sdrb_dense& scores, const sdrb_winners_spec& spec, const int32_t* ids, const float* grad_weights,
                        const sdrb_dense& out, hipStream_t stream) {
    const uint32_t n_ids = (uint32_t)scores.n_cols;
    return with_type(scores.type, [&](auto t) {
        return with_type(out.type, [&](auto o) {
            using T = decltype(t);
            using O = decltype(o);
            const size_t lds = (size_t)n_ids * sizeof(double);
            SDRB_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&k_winners_grad<T, O>), hipFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)lds));
            hipLaunchKernelGGL((k_winners_grad<T, O>), dim3((uint32_t)scores.n_rows), dim3(kThreads), lds, stream,
                               static_cast<const T*>(scores.data), scores.ld, n_ids, spec, ids, grad_weights, static_cast<O*>(out.data),
                               out.ld);
            SDRB_HIP(hipGetLastError());
            return SDRB_OK;
        });
    });
}

}  // namespace sdrb
