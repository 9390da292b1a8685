// The experts of each token and their weights, from the router's logits (kernels/router_topk.cuh: softmax and top-k, a thread block a token): scores,
// a bias for balance, groups of experts, the topk largest choices, renormalised weights.
//
// A warp has a token.  Its lanes hold the token's experts in registers, a group's experts in 32 / G neighbouring lanes (G the power of two at
// or above the groups), so that all groups find their best by the same few shuffles.  Choices are compared as 64-bit whole numbers that have
// the order of fp64 scores; the topk largest are taken one after the other by the warp's integer maximum (three redux instructions: upper and
// lower half, then the lowest index among equals).  Memory is a few hundred bytes a token: what bounds the kernel are its instructions, and
// the chain of topk maxima for a few tokens.
//
// Scores are fp64 because choices lie close to one another: with 256 experts and 4096 tokens some fp32 scores are within a rounding of the next one,
// and which expert a token gets must not depend on the exponential's last bit.
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
    const bool by_logit = !a.sigmoid && !a.bias && !a.sum2;
    float x[EPL];
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < EPL; i++) {
        const int m = sub + i * lanes;
        x[i] = group < a.groups && m < a.members ? logit(widen(row[e0 + m])) : -INFINITY;
        top = fmaxf(top, x[i]);
    }
    if (!a.sigmoid) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (top == -INFINITY) top = 0.f;           // then every exponential is 0
    }
    double total = 0.0;
    uint64_t key[EPL];
    if (by_logit) {                                // the order of the logits is that of the scores
#pragma unroll
        for (int i = 0; i < EPL; i++) {
            if (!a.renormalise) total += exp((double)x[i] - (double)top);
            key[i] = ordered((double)x[i]);
        }
        if (!a.renormalise) total = warp_sum(total);
    } else {
        double s[EPL];
#pragma unroll
        for (int i = 0; i < EPL; i++) {
            s[i] = a.sigmoid ? 1.0 / (1.0 + exp(-(double)x[i])) : exp((double)x[i] - (double)top);
            total += s[i];
        }
        if (!a.sigmoid) {
            total = warp_sum(total);
            if (total > 0.0) {
#pragma unroll
                for (int i = 0; i < EPL; i++) s[i] = s[i] / total;
            }
        }
#pragma unroll
        for (int i = 0; i < EPL; i++) {
            const int m = sub + i * lanes;
            const double b = a.bias && group < a.groups && m < a.members ? (double)a.bias[e0 + m] : 0.0;
            key[i] = ordered(s[i] + b);
        }
    }
#pragma unroll
    for (int i = 0; i < EPL; i++)                  // places that hold no expert come after all others
        if (group >= a.groups || sub + i * lanes >= a.members) key[i] = 0;

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
        const uint64_t score = group >= a.groups ? 0 : a.sum2 ? ordered(unordered(best) + unordered(second)) : best;
        int ahead = 0;                             // groups in front of this one
        for (int g = 0; g < a.groups; g++) {
            const uint64_t other = __shfl_sync(0xffffffffu, score, g << a.lanes_log2);
            ahead += other > score || (other == score && g < group);
        }
        if (ahead >= a.topk_groups) {
#pragma unroll
            for (int i = 0; i < EPL; i++) key[i] = 0;
        }
    }

    int mine = 0;                                  // lane k: the k-th expert
    uint64_t best = 0;
    int at = 0;
    auto find = [&]() {
        best = key[0]; at = 0;
#pragma unroll
        for (int i = 1; i < EPL; i++)
            if (key[i] > best) { best = key[i]; at = i; }
    };
    find();
    for (int k = 0; k < a.topk; k++) {
        const uint32_t hi = (uint32_t)(best >> 32), top_hi = __reduce_max_sync(0xffffffffu, hi);
        const uint32_t lo = hi == top_hi ? (uint32_t)best : 0u, top_lo = __reduce_max_sync(0xffffffffu, lo);
        const int e = e0 + sub + at * lanes;
        const int winner = (int)__reduce_min_sync(0xffffffffu, hi == top_hi && lo == top_lo ? (unsigned)e : 0xffffffffu);
        if (lane == k) mine = winner;
        if (e == winner) {
#pragma unroll
            for (int i = 0; i < EPL; i++)
                if (i == at) key[i] = 0;
            find();
        }
    }
    double w = 0.0;
    if (lane < a.topk) {
        const double v = (double)logit(widen(row[mine]));
        if (a.sigmoid) w = 1.0 / (1.0 + exp(-v));
        else {
            w = exp(v - (double)top);
            if (total > 0.0) w /= total;           // (0: none was taken, because weights are renormalised)
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
