// Norms and rotary positions of a step's queries and keys in one kernel (kernels/rope.cuh and the norms of queries and keys are kernels of their own in
// the graphs): every element is read and written once, which bounds the kernel for many tokens; a few tokens are bound by latency.
//
// Angles: position * frequency modulo a turn, in whole numbers.  A pair's frequency is kept in units of 2^-64 turn, the product wraps where turns
// do, and its upper 32 bits, taken as a signed number, are the angle in half a turn's 2^-31: cosine and sine are of an argument in [-1, 1)
// half turns whatever the position.  In fp32 the angle of token 131072 would have lost all bits below 2^-7.
#pragma once
#include <cmath>
#include "common.cuh"
#include "rows.cuh"

namespace w4a8 {
namespace rope {

constexpr int MAX_DIM = 256;

struct Args {
    const uint64_t *turns;
    const float *qw, *kw;
    const int32_t *position;
    const void *q, *k;
    void *q_out, *k_out;
    int64_t ldq, ldk, ldqo, ldko;
    float magnitude, inv_dim, eps;
    int heads_q, heads, dim, rotary, interleaved, variant, per_cta;       // heads: of queries and keys; per_cta of them to a CTA
    int skip_q, skip_k;                                                   // elements that are not turned already lie where they belong
};

// A group of LPH lanes has a head, a lane 8 elements of it: two runs of four at `a` and `b`, which hold four whole pairs where the head is
// rotated (i and i + rotary / 2 side by side in one lane) and eight neighbours elsewhere.  A CTA has one token's heads, so that
// cosines and sines are computed once for all of them.
constexpr int THREADS = 128, BATCH = 4;                                   // BATCH heads' loads of a lane in flight

template <typename T, int LPH>
__global__ void __launch_bounds__(THREADS) rope_kernel(const Args a) {
    __shared__ float2 turn[MAX_DIM / 2];
    const int t = blockIdx.x, half = a.rotary / 2;
    pdl_wait();
    pdl_launch_dependents();
    const int pos = a.position[t];
    if (pos < 0) return;
    const int group = threadIdx.x / LPH, j = threadIdx.x % LPH;
    constexpr int GROUPS = THREADS / LPH;
    const bool turned = 8 * j < a.rotary, live = 8 * j < a.dim;
    const int ia = turned && !a.interleaved ? 4 * j : 8 * j, ib = turned && !a.interleaved ? 4 * j + half : 8 * j + 4;
    const int first = blockIdx.y * a.per_cta, last = min(first + a.per_cta, a.heads);
    const T *q = static_cast<const T *>(a.q) + (size_t)t * a.ldq, *k = static_cast<const T *>(a.k) + (size_t)t * a.ldk;
    T *qo = static_cast<T *>(a.q_out) + (size_t)t * a.ldqo, *ko = static_cast<T *>(a.k_out) + (size_t)t * a.ldko;
    float x[BATCH][8];
    auto fetch = [&](int h0) {
#pragma unroll
        for (int b = 0; b < BATCH; b++) {
            const int h = h0 + b * GROUPS;
#pragma unroll
            for (int i = 0; i < 8; i++) x[b][i] = 0.f;
            if (h < last && live) {
                const bool is_q = h < a.heads_q;
                const T *src = is_q ? q + (size_t)h * a.dim : k + (size_t)(h - a.heads_q) * a.dim;
                if (turned || !(is_q ? a.skip_q : a.skip_k)) {
                    float lo[4], hi[4];
                    load_row<T, 4>(src + ia, lo);
                    load_row<T, 4>(src + ib, hi);
#pragma unroll
                    for (int i = 0; i < 4; i++) { x[b][i] = lo[i]; x[b][4 + i] = hi[i]; }
                }
            }
        }
    };
    fetch(first + group);
    for (int i = threadIdx.x; i < half; i += THREADS) {
        const uint64_t angle = (uint64_t)(uint32_t)pos * a.turns[i];
        float s, c;
        sincospif((float)(int32_t)(angle >> 32) * 0x1p-31f, &s, &c);
        turn[i] = make_float2(c * a.magnitude, s * a.magnitude);
    }
    __syncthreads();
    float c[4], s[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 cs = turned ? turn[4 * j + i] : make_float2(1.f, 0.f);
        c[i] = cs.x; s[i] = cs.y;
    }
    for (int h0 = first + group; h0 - group < last; h0 += BATCH * GROUPS) {
        if (h0 != first + group) fetch(h0);
#pragma unroll
        for (int b = 0; b < BATCH; b++) {
            const int h = h0 + b * GROUPS;
            if (h - group >= last) break;                                 // the same for the whole CTA: lanes of a group meet in the sums below
            const bool is_q = h < a.heads_q;
            if (a.variant != W4A8_NORM_NONE) {
                float ss = 0.f;
#pragma unroll
                for (int i = 0; i < 8; i++) ss = fmaf(x[b][i], x[b][i], ss);
#pragma unroll
                for (int o = 1; o < LPH; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                const float r = rsqrtf(fmaf(ss, a.inv_dim, a.eps));
                float lo[4] = {1.f, 1.f, 1.f, 1.f}, hi[4] = {1.f, 1.f, 1.f, 1.f};
                if (a.variant != W4A8_NORM_NO_SCALE && live) {
                    const float *w = is_q ? a.qw : a.kw;
                    load_row<float, 4>(w + ia, lo);
                    load_row<float, 4>(w + ib, hi);
                }
                const float one = a.variant == W4A8_NORM_ONE_PLUS ? 1.f : 0.f;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    x[b][i] = x[b][i] * r * (one + lo[i]);
                    x[b][4 + i] = x[b][4 + i] * r * (one + hi[i]);
                }
            }
            if (h < last && live && (turned || !(is_q ? a.skip_q : a.skip_k))) {
                float lo[4], hi[4];
                if (!turned || !a.interleaved) {                          // c = 1, s = 0 where nothing is turned
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        lo[i] = turned ? x[b][i] * c[i] - x[b][4 + i] * s[i] : x[b][i];
                        hi[i] = turned ? x[b][4 + i] * c[i] + x[b][i] * s[i] : x[b][4 + i];
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float u = x[b][2 * i] * c[i] - x[b][2 * i + 1] * s[i], v = x[b][2 * i + 1] * c[i] + x[b][2 * i] * s[i];
                        (i < 2 ? lo : hi)[2 * i & 3] = u;
                        (i < 2 ? lo : hi)[(2 * i & 3) + 1] = v;
                    }
                }
                T *dst = is_q ? qo + (size_t)h * a.dim : ko + (size_t)(h - a.heads_q) * a.dim;
                store_row<T, 4>(dst + ia, lo);
                store_row<T, 4>(dst + ib, hi);
            }
        }
    }
}

template <typename T, int LPH>
inline int launch_l(Args a, int T_rows, cudaStream_t st) {
    constexpr int GROUPS = THREADS / LPH;
    // a CTA takes one head a group while that leaves SMs idle, up to all of a token's heads where there are tokens enough for every SM
    const int passes = (a.heads + GROUPS - 1) / GROUPS;
    int per = 1;
    while (per < passes && (long)T_rows * ((passes + per - 1) / per) > 8L * sm_count()) per++;
    a.per_cta = per * GROUPS;
    const cudaError_t e = launch_pdl(rope_kernel<T, LPH>, dim3(T_rows, (a.heads + a.per_cta - 1) / a.per_cta), dim3(THREADS), 0, st, a);
    if (e != cudaSuccess) return cuda_fail(e, "rope launch");
    return launch_status("rope");
}
template <typename T>
inline int launch_t(const Args &a, int T_rows, cudaStream_t st) {
    if (a.dim <= 64) return launch_l<T, 8>(a, T_rows, st);
    if (a.dim <= 128) return launch_l<T, 16>(a, T_rows, st);
    return launch_l<T, 32>(a, T_rows, st);
}
inline int launch(const Args &a, int T_rows, int dtype, cudaStream_t st) {
    if (dtype == W4A8_F32) return launch_t<float>(a, T_rows, st);
    return dtype == W4A8_F16 ? launch_t<__half>(a, T_rows, st) : launch_t<__nv_bfloat16>(a, T_rows, st);
}

// Frequencies in units of 2^-64 turn.  long double has the 64 bits that they are kept in.
inline bool table(int rotary, double base, int scaling, double factor, double original, double low, double high, const double *divisor, uint64_t *turns, float *magnitude) {
    const long double two_pi = 2.0L * 3.14159265358979323846264338327950288L;
    *magnitude = 1.0f;
    long double b = base;
    if (scaling == W4A8_ROPE_NTK && rotary > 2) b = base * powl(factor, (long double)rotary / (rotary - 2));
    long double first = 0, last = 0;
    if (scaling == W4A8_ROPE_YARN) {
        const auto at = [&](long double n) { return rotary * logl(original / (n * two_pi)) / (2 * logl(b)); };
        first = fmaxl(0, floorl(at(high > 0 ? high : 32)));
        last = fminl(rotary - 1, ceill(at(low > 0 ? low : 1)));
        if (factor > 1) *magnitude = (float)(0.1L * logl(factor) + 1);
    }
    for (int i = 0; i < rotary / 2; i++) {
        long double f = powl(b, -2.0L * i / rotary);
        if (scaling == W4A8_ROPE_LINEAR) f /= factor;
        if (scaling == W4A8_ROPE_DIVISORS) f /= divisor[i];
        if (scaling == W4A8_ROPE_YARN) {
            const long double ramp = fminl(1, fmaxl(0, (i - first) / fmaxl(last - first, 1e-3L)));
            f *= 1 - ramp + ramp / factor;
        }
        if (scaling == W4A8_ROPE_BANDS) {
            const long double l = low > 0 ? low : 1, h = high > 0 ? high : 4;
            const long double ramp = fminl(1, fmaxl(0, (original * f / two_pi - l) / (h - l)));
            f *= ramp + (1 - ramp) / factor;
        }
        const long double turn = f / two_pi;
        if (!(turn >= 0) || turn > 1e15L) return false;
        const long double part = turn - floorl(turn);
        turns[i] = (uint64_t)fminl(roundl(part * 0x1p64L), 0x1.fffffffffffffffep63L);
    }
    return true;
}

}  // namespace rope
}  // namespace w4a8
