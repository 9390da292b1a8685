// Norms and rotary positions of a step's queries and keys in one kernel (kernels/rope.cuh and the norms of queries and keys are kernels of their own in
// the graphs): every element is read and written once, which bounds the kernel for many tokens; a few tokens are bound by latency.
//
// Angles: position * frequency modulo a turn, in whole numbers.  A pair's frequency is kept in units of 2^-64 turn, the product wraps where turns
// do, and its upper 32 bits, taken as a signed number, are the angle in half a turn's 2^-31: cosine and sine are of an argument in [-1, 1)
// half turns whatever the position.  In fp32 the angle of token 131072 would have lost all bits below 2^-7.
#pragma once
#include <cmath>
#include <type_traits>
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
    double eps64;
    float magnitude, inv_dim, eps;
    int heads_q, heads, dim, rotary, interleaved, variant, per_cta;       // heads: of queries and keys; per_cta of them to a CTA
    int skip_q, skip_k;                                                   // elements that are not turned already lie where they belong
};

// A group of LPH lanes has a head, a lane two runs of V of its elements, at `ia` and `ib`: V whole pairs where the head is rotated (i and
// i + rotary / 2 in one lane) and neighbours elsewhere.  A run is 16 bytes (V 4 of fp32, 8 of 16 bits; 4 there too where rotary / 2 is no
// multiple of 8, dim none of 16, or weights come with it).  A CTA has one token's heads, so that cosines and sines are computed once for all of them.
//
// Many tokens: bytes in flight are the bound, since each CTA waits for its position, then its rows, then stores.  Rows are asked for at once, before the
// position is known, BATCH heads a lane.  8000 tokens of 40 heads of 128 in bf16, half of them turned, 28 us: 5.8 TB/s; rows held widened while in
// flight, and so fewer CTAs, 46.
// Threads of a CTA: 40 heads divide into groups of eight and not of sixteen, and smaller CTAs wait for less at their barrier (8000 tokens in bf16, 128 threads / 64: 29.3 / 28.0 us,
// with norms 38.6 / 36.4); fp32 rows, whose loads fill the registers, lose by it (52.2 / 55.1).
template <typename T> constexpr int CTA = sizeof(T) == 4 ? 128 : 64;

// A head's factor comes from a sum of up to 256 squares in fp32, eps rounded to it and a reciprocal root within 2 ulp: within 2^-20 of itself where fp32 holds the squares, which it does
// for factors between these two (2^-60, 2^40) and always for fp16 elements.  Heads of elements around 2e18 and above, or of tiny ones beside no eps, are summed again in fp64 before anything of their batch is stored, since
// outputs may lie on inputs.  All sums of a batch first: looked at head by head, in between the stores, 8000 tokens with weighted norms took 5 to 11 % longer.
constexpr uint32_t FACTOR_MIN = 0x21800000u, FACTOR_MAX = 0x53800000u;
__device__ __forceinline__ uint32_t outside(float r) { return __float_as_uint(r) - FACTOR_MIN; }          // above FACTOR_MAX - FACTOR_MIN: outside, infinite or not a number

template <typename T, int V, int LPH, int BATCH>                         // BATCH heads' loads of a lane in flight
__global__ void __launch_bounds__(CTA<T>) rope_kernel(const Args a) {
    constexpr bool WIDE = !std::is_same<T, __half>::value;
    __shared__ float2 turn[MAX_DIM / 2];
    const int t = blockIdx.x, half = a.rotary / 2;
    const int group = threadIdx.x / LPH, j = threadIdx.x % LPH;
    constexpr int THREADS = CTA<T>, GROUPS = THREADS / LPH;
    const bool turned = 2 * V * j < a.rotary, live = 2 * V * j < a.dim;
    const int ia = turned && !a.interleaved ? V * j : 2 * V * j, ib = turned && !a.interleaved ? V * j + half : 2 * V * j + V;
    const int first = blockIdx.y * a.per_cta, last = min(first + a.per_cta, a.heads);
    const T *q = static_cast<const T *>(a.q) + (size_t)t * a.ldq, *k = static_cast<const T *>(a.k) + (size_t)t * a.ldk;
    T *qo = static_cast<T *>(a.q_out) + (size_t)t * a.ldqo, *ko = static_cast<T *>(a.k_out) + (size_t)t * a.ldko;
    pdl_wait();
    pdl_launch_dependents();
    Packed<T, V> raw[BATCH][2];
    auto fetch = [&](int h0) {
#pragma unroll
        for (int b = 0; b < BATCH; b++) {
            const int h = h0 + b * GROUPS;
            raw[b][0].clear();
            raw[b][1].clear();
            if (h < last && live) {
                const bool is_q = h < a.heads_q;
                const T *src = is_q ? q + (size_t)h * a.dim : k + (size_t)(h - a.heads_q) * a.dim;
                if (turned || !(is_q ? a.skip_q : a.skip_k)) {
                    raw[b][0].load(src + ia);
                    raw[b][1].load(src + ib);
                }
            }
        }
    };
    fetch(first + group);
    const int pos = a.position[t];
    if (pos < 0) return;
    for (int i = threadIdx.x; i < half; i += THREADS) {
        const uint64_t angle = (uint64_t)(uint32_t)pos * a.turns[i];
        float s, c;
        sincospif((float)(int32_t)(angle >> 32) * 0x1p-31f, &s, &c);
        turn[i] = make_float2(c * a.magnitude, s * a.magnitude);
    }
    __syncthreads();
    const float2 *mine = turn + V * j;                                    // this lane's pairs
    const auto factor = [&](const float (&u)[V], const float (&v)[V]) {   // lanes of a group meet here
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < V; i++) ss = fmaf(u[i], u[i], fmaf(v[i], v[i], ss));
#pragma unroll
        for (int o = 1; o < LPH; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        return rsqrtf(fmaf(ss, a.inv_dim, a.eps));
    };
    for (int h0 = first + group; h0 - group < last; h0 += BATCH * GROUPS) {
        if (h0 != first + group) fetch(h0);
        float r[BATCH];
        if (WIDE && a.variant != W4A8_NORM_NONE) {
            uint32_t worst = 0;
#pragma unroll
            for (int b = 0; b < BATCH; b++) {
                float u[V], v[V];
                raw[b][0].unpack(u);
                raw[b][1].unpack(v);
                r[b] = factor(u, v);
                if (h0 + b * GROUPS < last) worst = max(worst, outside(r[b]));
            }
            if (__any_sync(0xffffffffu, worst > FACTOR_MAX - FACTOR_MIN)) {
#pragma unroll
                for (int b = 0; b < BATCH; b++) {
                    const int h = h0 + b * GROUPS;
                    const bool is_q = h < a.heads_q;
                    const T *src = is_q ? q + (size_t)h * a.dim : k + (size_t)(h - a.heads_q) * a.dim;
                    double ss = 0.0;
#pragma unroll 1
                    for (int i = 0; i < 2 * V && h < last && live; i++) {
                        const double x = (double)(float)src[i < V ? ia + i : ib + i - V];
                        ss = fma(x, x, ss);
                    }
#pragma unroll 1
                    for (int o = 1; o < LPH; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                    if (outside(r[b]) > FACTOR_MAX - FACTOR_MIN) r[b] = (float)rsqrt(ss / a.dim + a.eps64);
                }
            }
        }
#pragma unroll
        for (int b = 0; b < BATCH; b++) {
            const int h = h0 + b * GROUPS;
            if (h - group >= last) break;                                 // the same for the whole CTA
            const bool is_q = h < a.heads_q;
            float u[V], v[V];                                             // the two runs
            raw[b][0].unpack(u);
            raw[b][1].unpack(v);
            if (a.variant != W4A8_NORM_NONE) {
                if (!WIDE) r[b] = factor(u, v);
                if (a.variant != W4A8_NORM_NO_SCALE && live) {
                    const float *w = is_q ? a.qw : a.kw;
                    const float one = a.variant == W4A8_NORM_ONE_PLUS ? 1.f : 0.f;
                    float lo[V], hi[V];
                    load_row<float, V>(w + ia, lo);
                    load_row<float, V>(w + ib, hi);
#pragma unroll
                    for (int i = 0; i < V; i++) { u[i] = u[i] * r[b] * (one + lo[i]); v[i] = v[i] * r[b] * (one + hi[i]); }     // r may be near an end of fp32, where r * w is not one
                } else {
#pragma unroll
                    for (int i = 0; i < V; i++) { u[i] *= r[b]; v[i] *= r[b]; }
                }
            }
            if (h < last && live && (turned || !(is_q ? a.skip_q : a.skip_k))) {
                if (turned && !a.interleaved) {
#pragma unroll
                    for (int i = 0; i < V; i++) {
                        const float2 cs = mine[i];
                        const float w = u[i] * cs.x - v[i] * cs.y;
                        v[i] = v[i] * cs.x + u[i] * cs.y;
                        u[i] = w;
                    }
                } else if (turned) {
#pragma unroll
                    for (int i = 0; i < V; i += 2) {
                        const float2 cs = mine[i / 2], ds = mine[(V + i) / 2];
                        const float w = u[i] * cs.x - u[i + 1] * cs.y, z = v[i] * ds.x - v[i + 1] * ds.y;
                        u[i + 1] = u[i + 1] * cs.x + u[i] * cs.y;
                        v[i + 1] = v[i + 1] * ds.x + v[i] * ds.y;
                        u[i] = w;
                        v[i] = z;
                    }
                }
                T *dst = is_q ? qo + (size_t)h * a.dim : ko + (size_t)(h - a.heads_q) * a.dim;
                store_row<T, V>(dst + ia, u);
                store_row<T, V>(dst + ib, v);
            }
        }
    }
}

template <typename T, int V, int LPH>
inline int launch_l(Args a, int T_rows, cudaStream_t st) {
    constexpr int THREADS = CTA<T>, GROUPS = THREADS / LPH;
    // a CTA takes one head a group while that leaves SMs idle, up to all of a token's heads where there are tokens enough for every SM
    const int passes = (a.heads + GROUPS - 1) / GROUPS;
    int per = 1;
    while (per < passes && (long)T_rows * ((passes + per - 1) / per) > 8L * sm_count()) per++;
    a.per_cta = per * GROUPS;
    const dim3 grid(T_rows, (a.heads + a.per_cta - 1) / a.per_cta);
    constexpr int MOST = V == 8 ? 3 : 5;
    const cudaError_t e = per == 1 ? launch_pdl(rope_kernel<T, V, LPH, 1>, grid, dim3(THREADS), 0, st, a)
                                   : launch_pdl(rope_kernel<T, V, LPH, MOST>, grid, dim3(THREADS), 0, st, a);
    if (e != cudaSuccess) return cuda_fail(e, "rope launch");
    return launch_status("rope");
}
template <typename T, int V>
inline int launch_v(const Args &a, int T_rows, cudaStream_t st) {
    if (a.dim <= 8 * V) return launch_l<T, V, 4>(a, T_rows, st);
    if (a.dim <= 16 * V) return launch_l<T, V, 8>(a, T_rows, st);
    if (a.dim <= 32 * V || V == 8) return launch_l<T, V, 16>(a, T_rows, st);
    return launch_l<T, V, V == 4 ? 32 : 16>(a, T_rows, st);
}
template <typename T>
inline int launch_16(const Args &a, int T_rows, cudaStream_t st) {
    // Runs of 8 where pairs and heads allow, but with weights, which are read for each head and twice as wide as the elements, 4: 8000 tokens of 40 heads of 128
    // with weighted norms 43.9 us in runs of 8, 38.7 in runs of 4 (interleaved 57.4 and 41.1); without weights 36.0 and more.
    const bool weighted = a.variant == W4A8_NORM_SCALE || a.variant == W4A8_NORM_ONE_PLUS;
    return a.dim % 16 == 0 && a.rotary % 16 == 0 && !weighted ? launch_v<T, 8>(a, T_rows, st) : launch_v<T, 4>(a, T_rows, st);
}
inline int launch(const Args &a, int T_rows, int dtype, cudaStream_t st) {
    if (dtype == W4A8_F32) return launch_v<float, 4>(a, T_rows, st);
    return dtype == W4A8_F16 ? launch_16<__half>(a, T_rows, st) : launch_16<__nv_bfloat16>(a, T_rows, st);
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
