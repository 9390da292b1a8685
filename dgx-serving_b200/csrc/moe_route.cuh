// The experts of each token and their weights, from the router's logits (kernels/router_topk.cuh: softmax and top-k, a thread block a token): scores,
// a bias for balance, groups of experts, the topk largest choices, renormalised weights.
//
// A warp has a token.  Its lanes hold the token's experts in registers, a group's experts in 32 / G neighbouring lanes (G the power of two at
// or above the groups), so that all groups find their best by the same few shuffles.  The topk largest choices are taken one after the other by the
// warp's integer maximum of numbers in the order of the choices, and the lowest index among equals.  Memory is a few hundred bytes a token: what
// bounds the kernel are its instructions, and the chain of topk maxima for a few tokens.
//
// Choices lie close to one another: with 256 experts and 4096 tokens some fp32 scores are within a rounding of the next one, and which expert a
// token gets must not depend on the exponential's last bit.  They are compared in fp64, then; but a token whose fp32 choices are further apart
// than fp32 can be wrong (all but a few in a thousand) has the same order in both and is done with 32-bit maxima.  4096 tokens of 256 experts in 8 groups,
// sigmoid and bias: 16.6 us all in fp64.
#pragma once
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
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float warp_max(float v) {                // of numbers that are not negative
    return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v)));
}
// The warp's largest key, and the lowest expert that has it.
__device__ __forceinline__ uint32_t take(uint32_t best, int e, uint32_t &top) {
    top = __reduce_max_sync(0xffffffffu, best);
    return __reduce_min_sync(0xffffffffu, best == top ? (uint32_t)e : 0xffffffffu);
}
__device__ __forceinline__ uint32_t take(uint64_t best, int e, uint64_t &top) {
    const uint32_t hi = (uint32_t)(best >> 32), top_hi = __reduce_max_sync(0xffffffffu, hi);
    const uint32_t lo = hi == top_hi ? (uint32_t)best : 0u, top_lo = __reduce_max_sync(0xffffffffu, lo);
    top = (uint64_t)top_hi << 32 | top_lo;
    return __reduce_min_sync(0xffffffffu, best == top ? (uint32_t)e : 0xffffffffu);
}
__device__ __forceinline__ double number(uint64_t k) { return unordered(k); }
__device__ __forceinline__ float number(uint32_t k) { return unordered(k); }

// The topk largest of the warp's keys (0: no expert there); lane k gets the k-th expert.  slack: what the difference of two choices may be wrong
// by; < 0: nothing, equal keys are equal choices.  False: the keys do not decide.
template <typename KEY, int EPL>
__device__ __forceinline__ bool select(const Args &a, KEY (&key)[EPL], int group, int lane, int e_first, int lanes, float slack, int &mine) {
    const bool loose = slack >= 0.f;
    bool sure = true;
    if (a.topk_groups < a.groups) {
        KEY best = 0, second = 0;
#pragma unroll
        for (int i = 0; i < EPL; i++) {
            second = max(second, min(best, key[i]));
            best = max(best, key[i]);
        }
        for (int o = 1; o < lanes; o <<= 1) {
            const KEY b2 = __shfl_xor_sync(0xffffffffu, best, o), s2 = __shfl_xor_sync(0xffffffffu, second, o);
            second = max(max(second, s2), min(best, b2));
            best = max(best, b2);
        }
        const KEY score = group >= a.groups ? 0 : a.sum2 ? ordered(number(best) + number(second)) : best;
        int ahead = 0;                             // groups in front of this one
        bool close = false;
        for (int g = 0; g < a.groups; g++) {
            const KEY other = __shfl_sync(0xffffffffu, score, g << a.lanes_log2);
            ahead += other > score || (other == score && g < group);
            if (loose) close |= g != group && !(fabsf((float)number(other) - (float)number(score)) > 2.f * slack);
        }
        // (a group next to another one matters where one of the two is taken and the other is not: looked at for all that are next to the border)
        if (loose) sure = !__any_sync(0xffffffffu, close && group < a.groups && (ahead == a.topk_groups || ahead == a.topk_groups - 1));
        if (ahead >= a.topk_groups) {
#pragma unroll
            for (int i = 0; i < EPL; i++) key[i] = 0;
        }
    }
    KEY best = 0;
    int at = 0;
    auto find = [&]() {
        best = key[0]; at = 0;
#pragma unroll
        for (int i = 1; i < EPL; i++)
            if (key[i] > best) { best = key[i]; at = i; }
    };
    find();
    KEY before = 0;
    for (int k = 0; k < a.topk + (loose ? 1 : 0); k++) {
        const int e = e_first + at * lanes;
        KEY top;
        const int winner = (int)take(best, e, top);
        if (loose && k > 0 && top != 0 && !(number(before) - number(top) > slack)) sure = false;
        before = top;
        if (k == a.topk) break;
        if (lane == k) mine = winner;
        if (e == winner) {
#pragma unroll
            for (int i = 0; i < EPL; i++)
                if (i == at) key[i] = 0;
            find();
        }
    }
    return sure;
}

constexpr int WARPS = 4;

template <typename T, int EPL>                     // EPL experts a lane
__global__ void __launch_bounds__(WARPS * 32) route_kernel(const Args a) {
    const int lane = threadIdx.x & 31;
    const long t = (long)blockIdx.x * WARPS + (threadIdx.x >> 5);
    pdl_wait();
    pdl_launch_dependents();
    if (t >= a.S) return;
    const T *row = static_cast<const T *>(a.logits) + t * a.ld;
    const int lanes = 1 << a.lanes_log2, group = lane >> a.lanes_log2, sub = lane & (lanes - 1);
    const int e0 = group * a.members;              // expert i of this lane is e0 + sub + i * lanes
    const auto there = [&](int i) { return group < a.groups && sub + i * lanes < a.members; };
    const bool by_logit = !a.sigmoid && !a.bias && !a.sum2;
    float x[EPL];
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < EPL; i++) {
        x[i] = there(i) ? logit(widen(row[e0 + sub + i * lanes])) : -INFINITY;
        top = fmaxf(top, x[i]);
    }
    if (!a.sigmoid) {
        top = unordered(__reduce_max_sync(0xffffffffu, ordered(top)));
        if (top == -INFINITY) top = 0.f;           // then every exponential is 0
    }
    int mine = 0;                                  // lane k: the k-th expert
    bool sure;
    {
        uint32_t key[EPL];
        float slack = -1.f;
        if (by_logit) {                            // the order of the logits is that of the scores
#pragma unroll
            for (int i = 0; i < EPL; i++) key[i] = there(i) ? ordered(x[i]) : 0u;
        } else {
            float s[EPL], sum = 0.f, largest = 0.f;
#pragma unroll
            for (int i = 0; i < EPL; i++) {
                s[i] = a.sigmoid ? 1.f / (1.f + expf(-x[i])) : expf(x[i] - top);
                sum += s[i];
            }
            if (!a.sigmoid) {
                sum = warp_sum(sum);
                const float inv = sum > 0.f ? 1.f / sum : 1.f;
#pragma unroll
                for (int i = 0; i < EPL; i++) s[i] *= inv;
            }
#pragma unroll
            for (int i = 0; i < EPL; i++) {
                const float b = a.bias && there(i) ? a.bias[e0 + sub + i * lanes] : 0.f;
                largest = fmaxf(largest, s[i] + fabsf(b));
                s[i] += b;
                largest = s[i] == s[i] && fabsf(s[i]) < INFINITY ? largest : INFINITY;
                key[i] = there(i) ? ordered(s[i]) : 0u;
            }
            // A score is off by at most 64 * 2^-24 of itself (the exponential 2 ulp, a sum of up to 1024 terms by 64 + 5 roundings of halves, a reciprocal and
            // a product), a choice by one rounding more, and two of them by twice that.
            slack = warp_max(largest) * 0x1p-16f;
        }
        sure = select(a, key, group, lane, e0 + sub, lanes, slack, mine);
        if (!by_logit && !(slack < INFINITY)) sure = false;
    }
    double total = 0.0;
    if (!a.sigmoid && (!sure || !a.renormalise)) {
#pragma unroll
        for (int i = 0; i < EPL; i++) total += exp((double)x[i] - (double)top);
        total = warp_sum(total);
    }
    if (!sure) {
        uint64_t key[EPL];
#pragma unroll
        for (int i = 0; i < EPL; i++) {
            double s = a.sigmoid ? 1.0 / (1.0 + exp(-(double)x[i])) : exp((double)x[i] - (double)top);
            if (!a.sigmoid && total > 0.0) s /= total;
            key[i] = there(i) ? ordered(s + (a.bias ? (double)a.bias[e0 + sub + i * lanes] : 0.0)) : 0ull;
        }
        select(a, key, group, lane, e0 + sub, lanes, -1.f, mine);
    }
    double w = 0.0;
    if (lane < a.topk) {
        const double v = (double)logit(widen(row[mine]));
        if (a.sigmoid) w = 1.0 / (1.0 + exp(-v));
        else {
            w = exp(v - (double)top);
            if (total > 0.0) w /= total;           // (0: not taken, because weights are renormalised)
        }
    }
    if (a.renormalise) {
        const double sum = warp_sum(w);
        if (sum > 0.0) w /= sum;
    }
    if (lane < a.topk) {
        a.idx[t * a.topk + lane] = mine;
        a.weight[t * a.topk + lane] = (float)(w * (double)a.scale);
    }
}

template <typename T>
inline int launch_t(const Args &a, cudaStream_t st) {
    const int epl = (a.members + (1 << a.lanes_log2) - 1) >> a.lanes_log2;
    const dim3 grid((unsigned)((a.S + (long)WARPS - 1) / WARPS)), block(WARPS * 32);
    cudaError_t e;
    if (epl <= 1) e = launch_pdl(route_kernel<T, 1>, grid, block, 0, st, a);
    else if (epl <= 2) e = launch_pdl(route_kernel<T, 2>, grid, block, 0, st, a);
    else if (epl <= 4) e = launch_pdl(route_kernel<T, 4>, grid, block, 0, st, a);
    else if (epl <= 8) e = launch_pdl(route_kernel<T, 8>, grid, block, 0, st, a);
    else if (epl <= 16) e = launch_pdl(route_kernel<T, 16>, grid, block, 0, st, a);
    else if (epl <= 32) e = launch_pdl(route_kernel<T, 32>, grid, block, 0, st, a);
    else e = launch_pdl(route_kernel<T, 64>, grid, block, 0, st, a);         // groups just above a power of two: 1024 / 17 experts on one lane
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
