// The experts of each token and their weights, from the router's logits (kernels/router_topk.cuh: softmax and top-k, a thread block a token): scores,
// a bias for balance, groups of experts, the topk largest choices, renormalised weights.
//
// A warp has a token.  Its lanes hold the token's experts in registers, a group's experts in 32 / G neighbouring lanes (G the power of two at
// or above the groups) and neighbours in a lane, so that all groups find their best by the same few shuffles and a lane's logits come by 16-byte loads.
// Each lane sorts what it holds, and the topk largest are taken
// from the lanes' heads one after the other, by two integer maxima over the warp: the fp32 choice in an order that whole numbers have, then the
// lowest index among equals.  Memory is a few hundred bytes a token: what bounds the kernel are its instructions, and for a few tokens the chain of maxima.
//
// Choices lie close to one another: with 256 experts and 4096 tokens some fp32 scores are within a rounding of the next one, and which expert a
// token gets must not depend on the exponential's last bit.  So four candidates more than topk are taken; where neighbours among them are closer than
// fp32 can be wrong (4 tokens in 100), the candidates are put in order by their choices in fp64, one a lane, and where that does not decide either
// (a border of groups, more near values than candidates) the whole token is done again in fp64.  There is a lane for 32 candidates, and of the next one its choice.
#pragma once
#include <type_traits>
#include "common.cuh"
#include "rows.cuh"

namespace w4a8 {
namespace route {

constexpr int MAX_EXPERTS = 1024, MAX_TOPK = 32, MAX_GROUPS = 32;

struct Args {
    const void *logits;
    const float *bias;
    int32_t *idx;
    float *weight;
    int64_t ld;
    int S, experts, topk, sigmoid, groups, topk_groups, sum2, renormalise;
    int members, lanes_log2;                       // experts of a group; log2 of the lanes that hold them
    int wide;                                      // lanes are full, and what they hold is aligned to 16 bytes
    float scale;
};

// Numbers in an order that unsigned whole numbers have; -0 is 0.
__device__ __forceinline__ uint64_t ordered(double v) {
    const long long b = __double_as_longlong(v + 0.0);
    return (uint64_t)(b < 0 ? ~b : b | (1ll << 63));
}
__device__ __forceinline__ double unordered(uint64_t k) {
    const long long b = (long long)k;
    return __longlong_as_double(b < 0 ? b & ~(1ll << 63) : ~b);
}
__device__ __forceinline__ float logit(float x) { return x != x ? -INFINITY : fminf(x, 3.402823466e38f); }
template <typename T> __device__ __forceinline__ float widen(T x) { return (float)x; }

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The same for fp32.
__device__ __forceinline__ uint32_t ordered(float v) {
    const int b = __float_as_int(v + 0.f);
    return (uint32_t)(b < 0 ? ~b : b | (1 << 31));
}
__device__ __forceinline__ float unordered(uint32_t k) { return __int_as_float((int)k < 0 ? (int)k & 0x7fffffff : (int)~k); }
// e^v = 2^(v log2 e), the exponent as a sum of two numbers: within 6 * 2^-24 of itself where it is normal (ex2.approx 2^-22, a product, the second number's
// part of the result), without expf's cases.  The sigmoids of 4096 tokens by expf and an IEEE division: 14.6 us as above, 13.4 by __expf.
__device__ __forceinline__ float exp_close(float v) {
    constexpr double LOG2_E = 1.4426950408889634;
    constexpr float L = (float)LOG2_E, L2 = (float)(LOG2_E - (double)L);
    v = fminf(fmaxf(v, -200.f), 100.f);                                // 0 and infinity
    const float p = v * L, q = fmaf(v, L2, fmaf(v, L, -p));
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(p));
    return e * fmaf(q, (float)(1.0 / LOG2_E), 1.f);
}
__device__ __forceinline__ float reciprocal(float v) {                 // 1 ulp
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float warp_max(float v) {                // of numbers that are not negative
    return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v)));
}
// The topk largest fp64 choices (0: no expert there); equal ones by the lowest index.  Lane k gets the k-th expert.
__device__ __forceinline__ uint32_t take(uint64_t best, int e, uint64_t &top) {
    const uint32_t hi = (uint32_t)(best >> 32), top_hi = __reduce_max_sync(0xffffffffu, hi);
    const uint32_t lo = hi == top_hi ? (uint32_t)best : 0u, top_lo = __reduce_max_sync(0xffffffffu, lo);
    top = (uint64_t)top_hi << 32 | top_lo;
    return __reduce_min_sync(0xffffffffu, best == top ? (uint32_t)e : 0xffffffffu);
}
template <int EPL>
__device__ __noinline__ int select_double(const Args &a, uint64_t (&key)[EPL], int group, int lane, int e0, int lanes) {
    uint64_t top;
    if (a.topk_groups < a.groups) {
        uint64_t best = 0, second = 0;
#pragma unroll
        for (int i = 0; i < EPL; i++) {
            second = max(second, min(best, key[i]));
            best = max(best, key[i]);
        }
        for (int o = 1; o < lanes; o <<= 1) {
            const uint64_t b2 = __shfl_xor_sync(0xffffffffu, best, o), s2 = __shfl_xor_sync(0xffffffffu, second, o);
            second = max(max(second, s2), min(best, b2));
            best = max(best, b2);
        }
        uint64_t score = group >= a.groups ? 0 : a.sum2 ? ordered(unordered(best) + unordered(second)) : best;
        bool open = false;
        for (int k = 0; k < a.topk_groups; k++)
            if ((int)take(score, group, top) == group) { open = true; score = 0; }
        if (!open) {
#pragma unroll
            for (int i = 0; i < EPL; i++) key[i] = 0;
        }
    }
    int mine = 0;
    for (int k = 0; k < a.topk; k++) {
        uint64_t best = key[0];
        int at = 0;
#pragma unroll
        for (int i = 1; i < EPL; i++)
            if (key[i] > best) { best = key[i]; at = i; }
        const int e = e0 + at, winner = (int)take(best, e, top);
        if (lane == k) mine = winner;
#pragma unroll
        for (int i = 0; i < EPL; i++)
            if (e == winner && i == at) key[i] = 0;
    }
    return mine;
}

// What a lane holds, as fp32 choice and index in one number (the index inverted, so that of equal choices the first is the largest), no two
// alike; 0 where there is none.  Up to eight are sorted once and then move up; more are looked
// through each time (4096 tokens of 512 experts, sixteen a lane, topk 8: 12.2 us so, 18.7 sorted).
template <int N>
struct Held {
    static constexpr bool SORTED = N <= 8;
    uint64_t key[N];
    __device__ __forceinline__ void settle() {
        if constexpr (SORTED) {                    // odd-even merge sort, largest first
#pragma unroll
            for (int p = 1; p < N; p <<= 1)
#pragma unroll
                for (int k = p; k >= 1; k >>= 1)
#pragma unroll
                    for (int j = k % p; j + k < N; j += 2 * k)
#pragma unroll
                        for (int i = 0; i < k; i++)
                            if (i + j + k < N && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
                                const uint64_t u = key[i + j], v = key[i + j + k];
                                key[i + j] = max(u, v);
                                key[i + j + k] = min(u, v);
                            }
        }
    }
    __device__ __forceinline__ uint64_t best() const {
        if constexpr (SORTED) return key[0];
        uint64_t m[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < N; i++) m[i & 3] = max(m[i & 3], key[i]);
        return max(max(m[0], m[1]), max(m[2], m[3]));
    }
    __device__ __forceinline__ uint32_t second(uint64_t first) const {           // the second choice, 0 if there is none
        if constexpr (SORTED) return N > 1 ? (uint32_t)(key[N > 1] >> 32) : 0u;
        uint64_t m = 0;
#pragma unroll
        for (int i = 0; i < N; i++) m = key[i] != first ? max(m, key[i]) : m;
        return (uint32_t)(m >> 32);
    }
    __device__ __forceinline__ void drop(uint64_t first, bool yes) {
        if constexpr (SORTED) {
#pragma unroll
            for (int i = 0; i + 1 < N; i++) key[i] = yes ? key[i + 1] : key[i];
            key[N - 1] = yes ? 0 : key[N - 1];
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) key[i] = yes && key[i] == first ? 0 : key[i];
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < N; i++) key[i] = 0;
    }
};

constexpr int WARPS = 4, SPARE = 4;

// EPL experts a lane.  BY_LOGIT: a softmax without a bias whose groups are not added up, where the order of the logits is that of the scores: nothing to
// be decided in fp64, and without that code 4096 tokens of 128 experts take 3.8 us and not 5.3.
template <typename T, int EPL, bool BY_LOGIT>
__global__ void __launch_bounds__(WARPS * 32) route_kernel(const Args a) {
    const int lane = threadIdx.x & 31;
    const long t = (long)blockIdx.x * WARPS + (threadIdx.x >> 5);
    pdl_wait();
    pdl_launch_dependents();
    if (t >= a.S) return;
    const T *row = static_cast<const T *>(a.logits) + t * a.ld;
    const int lanes = 1 << a.lanes_log2, group = lane >> a.lanes_log2, sub = lane & (lanes - 1);
    const int e0 = group * a.members + sub * EPL;  // the first expert of this lane
    const auto there = [&](int i) { return group < a.groups && sub * EPL + i < a.members; };
    // every load at once: places that hold no expert read the row's first
    float x[EPL], b[EPL];
    bool loaded = false;
    if constexpr (EPL % Row<T>::N == 0) {
        if (a.wide) {
            load_row<T, EPL>(row + (group < a.groups ? e0 : 0), x);
#pragma unroll
            for (int i = 0; i < EPL; i++) b[i] = 0.f;
            if (a.bias) load_row<float, EPL>(a.bias + (group < a.groups ? e0 : 0), b);
            loaded = true;
        }
    }
    if (!loaded) {
#pragma unroll
        for (int i = 0; i < EPL; i++) x[i] = widen(row[there(i) ? e0 + i : 0]);
#pragma unroll
        for (int i = 0; i < EPL; i++) b[i] = a.bias ? a.bias[there(i) ? e0 + i : 0] : 0.f;
    }
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < EPL; i++) {
        x[i] = there(i) ? logit(x[i]) : -INFINITY;
        top = fmaxf(top, x[i]);
    }
    if (!a.sigmoid) {
        top = unordered(__reduce_max_sync(0xffffffffu, ordered(top)));
        if (top == -INFINITY) top = 0.f;           // then every exponential is 0
    }
    Held<EPL> held;
    const auto hold = [&](int i, float c) { held.key[i] = there(i) ? (uint64_t)ordered(c) << 32 | ~(uint32_t)(e0 + i) : 0ull; };
    float slack = 0.f;
    if constexpr (BY_LOGIT) {
#pragma unroll
        for (int i = 0; i < EPL; i++) hold(i, x[i]);
    } else {
        float s[EPL], sum = 0.f, largest = 0.f;
#pragma unroll
        for (int i = 0; i < EPL; i++) {
            s[i] = a.sigmoid ? reciprocal(1.f + exp_close(-x[i])) : exp_close(x[i] - top);
            sum += s[i];
        }
        if (!a.sigmoid) {
            sum = warp_sum(sum);
            const float inv = sum > 0.f ? reciprocal(sum) : 1.f;
#pragma unroll
            for (int i = 0; i < EPL; i++) s[i] *= inv;
        }
#pragma unroll
        for (int i = 0; i < EPL; i++) {
            if (there(i)) largest = fmaxf(largest, s[i] + fabsf(b[i]));
            s[i] += b[i];
            largest = fabsf(s[i]) < INFINITY ? largest : INFINITY;
            hold(i, s[i]);
        }
        // How far a choice may be off, in units of 2^-24 of the largest score and bias together.  Sigmoid: exp_close 6, the sum 1, the reciprocal 2, the
        // bias 1: two choices 20, and 2^-19 is 32.  Softmax: exp_close 6 and its argument's rounding, |v| e^v < 0.4; a sum of up to 1024 terms 64 + 5; the
        // reciprocal 2; the product and the sum with the bias 2: two 160, and 2^-16 is 256.  And scores below 2^-126 are 0: four of them, in two sums of two, 2^-124.
        slack = warp_max(largest) * (a.sigmoid ? 0x1p-19f : 0x1p-16f) + 0x1p-124f;
    }
    held.settle();
    bool whole = !(slack < INFINITY);              // again in fp64
    if (a.topk_groups < a.groups) {
        const uint64_t first = held.best();
        uint32_t best = (uint32_t)(first >> 32), second = held.second(first);
        for (int o = 1; o < lanes; o <<= 1) {
            const uint32_t b2 = __shfl_xor_sync(0xffffffffu, best, o), s2 = __shfl_xor_sync(0xffffffffu, second, o);
            second = max(max(second, s2), min(best, b2));
            best = max(best, b2);
        }
        uint32_t score = group >= a.groups ? 0 : a.sum2 ? ordered(unordered(best) + unordered(second)) : best, before = 0;
        bool open = false;
        for (int k = 0; k < a.topk_groups + (BY_LOGIT ? 0 : 1); k++) { // the best group of those that are left, and of equal ones the first
            const uint32_t most = __reduce_max_sync(0xffffffffu, score), g = __reduce_min_sync(0xffffffffu, score == most ? (uint32_t)group : 0xffffffffu);
            if (k == a.topk_groups) whole |= !(unordered(before) - unordered(most) > 2.f * slack);      // the last group taken and the first that is not
            else if ((int)g == group) { open = true; score = 0; }
            before = most;
        }
        if (!open) held.clear();
    }
    const int wanted = BY_LOGIT ? a.topk : min(33, a.topk + SPARE);       // the 33rd has no lane, it is the best of those that are not taken
    int mine = 0, found = 0;                       // lane k: the k-th candidate
    uint32_t lowest = 0;
    float choice = 0.f;
    for (int k = 0; k < wanted; k++) {
        const uint64_t best = held.best();
        const uint32_t hi = (uint32_t)(best >> 32), top_hi = __reduce_max_sync(0xffffffffu, hi);
        if (top_hi == 0) break;
        lowest = top_hi;
        const uint32_t top_lo = __reduce_max_sync(0xffffffffu, hi == top_hi ? (uint32_t)best : 0u);
        if (lane == k) { mine = (int)~top_lo; choice = unordered(top_hi); }
        held.drop(best, hi == top_hi && (uint32_t)best == top_lo);
        found = k + 1;
    }
    if (!BY_LOGIT && !whole) {
        const float last = unordered(lowest), below = __shfl_down_sync(0xffffffffu, choice, 1), next = lane == 31 ? last : below;
        if (__any_sync(0xffffffffu, lane < a.topk && lane + 1 < found && !(choice - next > slack))) {
            // candidates that were not taken are further away than fp32 can be wrong, or there are none
            const float end = __shfl_sync(0xffffffffu, choice, a.topk - 1);
            if (found < wanted || end - last > slack) {
                const int lanes_taken = min(found, 32);
                double total = 1.0;
                if (!a.sigmoid) {
                    total = 0.0;
#pragma unroll
                    for (int i = 0; i < EPL; i++) total += exp((double)x[i] - (double)top);
                    total = warp_sum(total);
                }
                const double v = (double)logit(widen(row[mine]));
                double c = a.sigmoid ? 1.0 / (1.0 + exp(-v)) : exp(v - (double)top);
                if (!a.sigmoid && total > 0.0) c /= total;
                if (a.bias) c += (double)a.bias[mine];
                int ahead = 0, placed = 0;
                for (int k = 0; k < lanes_taken; k++) {
                    const double other = __shfl_sync(0xffffffffu, c, k);
                    const int e = __shfl_sync(0xffffffffu, mine, k);
                    ahead += other > c || (other == c && e < mine);
                }
                for (int k = 0; k < lanes_taken; k++) {
                    const int place = __shfl_sync(0xffffffffu, ahead, k), e = __shfl_sync(0xffffffffu, mine, k);
                    if (place == lane) placed = e;
                }
                mine = placed;
            } else whole = true;
        }
    }
    if (!BY_LOGIT && whole) {
        double total = 0.0;
        if (!a.sigmoid) {
#pragma unroll
            for (int i = 0; i < EPL; i++) total += exp((double)x[i] - (double)top);
            total = warp_sum(total);
        }
        uint64_t key[EPL];
#pragma unroll
        for (int i = 0; i < EPL; i++) {
            double s = a.sigmoid ? 1.0 / (1.0 + exp(-(double)x[i])) : exp((double)x[i] - (double)top);
            if (!a.sigmoid && total > 0.0) s /= total;
            key[i] = there(i) ? ordered(s + (double)b[i]) : 0ull;
        }
        mine = select_double(a, key, group, lane, e0, lanes);
    }
    // Weights in fp32.  Renormalised ones need the chosen scores up to a common factor alone, so the exponentials are of distances to the largest chosen logit:
    // the largest of all may belong to an expert that a bias or its group keeps out, and fp32 ends 104 below it.  Sigmoids below e^-64 are e^v to
    // 2^-92 of themselves, and get the same factor where all of the chosen are that small.  Scores below e^-745, which fp64 does not hold, are 0.
    // As a rule the largest of all is among the chosen (always, where the logits decide), as is a sigmoid that fp32 holds.
    constexpr float BARE = -64.f, LEAST = -745.f;
    float v = -INFINITY, w = 0.f;
    if (lane < a.topk) {
        v = logit(widen(row[mine]));
        w = a.sigmoid ? 1.f / (1.f + expf(-v)) : expf(v - top);
    }
    if constexpr (!BY_LOGIT) {
        const float first = a.sigmoid ? 0.f : top;
        const bool far = a.renormalise && !__any_sync(0xffffffffu, a.sigmoid ? v >= BARE : v == top);
        const float from = far ? unordered(__reduce_max_sync(0xffffffffu, ordered(v))) : first;
        if (far || (a.sigmoid && v < BARE)) w = v - first > LEAST ? expf(v - from) : 0.f;
    }
    float sum = warp_sum(w);
    if (!a.renormalise) {                          // softmax over all experts, the sum in fp32 as the weights are
        sum = 0.f;
        if (!a.sigmoid) {
#pragma unroll
            for (int i = 0; i < EPL; i++) sum += expf(x[i] - top);
            sum = warp_sum(sum);
        }
    }
    if (sum > 0.f) w /= sum;
    if (lane < a.topk) {
        a.idx[t * a.topk + lane] = mine;
        a.weight[t * a.topk + lane] = w * a.scale;
    }
}

template <typename T>
inline int launch_t(Args a, cudaStream_t st) {
    int epl = 1;
    while ((epl << a.lanes_log2) < a.members) epl *= 2;
    a.wide = a.members == epl << a.lanes_log2 && aligned(a.logits, 16) && a.ld * sizeof(T) % 16 == 0 && (!a.bias || aligned(a.bias, 16));
    const dim3 grid((unsigned)((a.S + (long)WARPS - 1) / WARPS)), block(WARPS * 32);
    const bool by_logit = !a.sigmoid && !a.bias && !a.sum2;
    const auto launch = [&](auto experts) {
        constexpr int N = decltype(experts)::value;
        return by_logit ? launch_pdl(route_kernel<T, N, true>, grid, block, 0, st, a) : launch_pdl(route_kernel<T, N, false>, grid, block, 0, st, a);
    };
    using std::integral_constant;
    cudaError_t e;
    if (epl <= 1) e = launch(integral_constant<int, 1>());
    else if (epl <= 2) e = launch(integral_constant<int, 2>());
    else if (epl <= 4) e = launch(integral_constant<int, 4>());
    else if (epl <= 8) e = launch(integral_constant<int, 8>());
    else if (epl <= 16) e = launch(integral_constant<int, 16>());
    else if (epl <= 32) e = launch(integral_constant<int, 32>());
    else e = launch(integral_constant<int, 64>());                       // groups just above a power of two: 1024 / 17 experts on one lane
    if (e != cudaSuccess) return cuda_fail(e, "moe_route launch");
    return launch_status("moe_route");
}
inline int launch(Args a, int dtype, cudaStream_t st) {
    int g = 1, log2 = 0;
    while (g < a.groups) { g *= 2; log2++; }
    a.members = a.experts / a.groups;
    a.lanes_log2 = 5 - log2;
    if (dtype == W4A8_F32) return launch_t<float>(a, st);
    return dtype == W4A8_F16 ? launch_t<__half>(a, st) : launch_t<__nv_bfloat16>(a, st);
}

}  // namespace route
}  // namespace w4a8
