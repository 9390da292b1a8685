// Residual add and norms of rows in one kernel, with the quantizer of the product that follows:
//   p = norm(y) * gate * alpha,  h' = h + p,  n = norm(h'),  n -> its own type and / or int8 codes.
// Each of these is a pass over the rows in the graphs (kernels/norm_fused.cuh, kernels/rmsnorm.cuh, kernels/quantize_x.cuh); together they read h and y
// once and write h' and n once, which is what bounds the kernel for many rows.  A CTA has a row, its threads keep the row's elements in registers
// between the passes over it: the sum of squares of y (if y is normed), the sum of squares of h', the largest magnitude of n (if a row has
// one scale).
//
// Every element is computed by single fp32 operations in a stated order and the sums of squares in fp64, with one rounding of the factor
// r to fp32: how many threads share a row, which S decides, then changes the order of the fp64 sum alone, and with it r by one fp32 step where r lies that near to
// the middle of two (one row in 10^8); all else is the same bits, and codes are the same wherever they are made.  One order for every cut, or a second and
// more exact sum near such a middle, costs registers that all rows pay for: 8192 x 5120 101 -> 120 us, 290 x 8192 4.15 -> 5.07.  The fp64
// additions cost nothing where HBM is the bound (one conversion and one fma an element, against 16 bytes of traffic).
#pragma once
#include "common.cuh"
#include "rows.cuh"

namespace w4a8 {
namespace addnorm {

constexpr int MAX_K = 32768;

struct Args {
    const void *h, *y;
    void *h_out, *n_out;
    const float *w, *pw, *gate;
    int64_t ldh, ldy, ldo, ldn, ldg;
    int8_t *xq;
    float *xs;
    int32_t *xsum;
    double inv_k, eps;
    float alpha;
    int K, variant, post, group;                  // group 32, or 0: one scale for the row
    int S;
};

// The sum over the CTA (WARP: over the warp), in every thread; the same bits in all of them.
template <bool WARP>
__device__ __forceinline__ double cta_sum(double v, double *sh) {
    const int lane = threadIdx.x & 31, warps = WARP ? 1 : blockDim.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (warps == 1) return v;
    if (lane == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < warps ? sh[lane] : 0.0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
template <bool WARP>
__device__ __forceinline__ float cta_max(float v, float *sh) {
    const int lane = threadIdx.x & 31, warps = WARP ? 1 : blockDim.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    if (warps == 1) return v;
    if (lane == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < warps ? sh[lane] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

template <int V>
__device__ __forceinline__ double squares(const float (&x)[V], double ss) {
#pragma unroll
    for (int i = 0; i < V; i++) ss = fma((double)x[i], (double)x[i], ss);
    return ss;
}
__device__ __forceinline__ bool takes_weight(int variant) { return variant == W4A8_NORM_SCALE || variant == W4A8_NORM_ONE_PLUS; }
// x * r * f, x * r * (1 + f) or x * r, from left to right.
template <int V>
__device__ __forceinline__ void normed(float (&x)[V], float r, const float (&f)[V], int variant) {
#pragma unroll
    for (int i = 0; i < V; i++) {
        x[i] = __fmul_rn(x[i], r);
        if (variant == W4A8_NORM_SCALE) x[i] = __fmul_rn(x[i], f[i]);
        if (variant == W4A8_NORM_ONE_PLUS) x[i] = __fmul_rn(x[i], __fadd_rn(1.f, f[i]));
    }
}

// Elements of one thread's vector: 16 bytes of rows where all are fp32, eight elements where some have 16 bits.
template <typename TH, typename TY>
constexpr int VEC = sizeof(TH) == 4 && sizeof(TY) == 4 ? 4 : 8;

// EP elements a thread.  EARLY: weights are asked for together with the rows and not behind the sums that they do not depend on: a
// trip to L2 less for each norm where a few rows are bound by latency (64 rows of 5120 with codes 3.3 -> 2.8 us), registers that cost CTAs where there are many.  SUM: there is a y.
// WARP: a row is one warp's, several rows a CTA's, and nothing is waited for: short rows in great number are otherwise bound by the rate at which CTAs start
// (8192 rows of 256 elements 8.9 us whatever is done to them, 4.5 to 5.6 so; above 512 elements sums of two rows are faster by CTAs, 8192 x 1024 20.4 and 21.3,
// and quantizers by warps, 8.9 and 8.2).
template <typename TH, typename TY, int EP, int MAXT, bool EARLY, bool SUM, bool WARP>
__global__ void __launch_bounds__(MAXT, 1) add_norm_kernel(const Args a) {
    constexpr int V = VEC<TH, TY>, NV = EP / V;
    __shared__ double sh_y[32], sh_h[32];
    __shared__ float sh_max[32];
    const int nt = WARP ? 32 : blockDim.x, tid = WARP ? threadIdx.x & 31 : threadIdx.x, nvec = a.K / V;
    const size_t row = WARP ? (size_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
    pdl_wait();
    pdl_launch_dependents();
    if (WARP && row >= (size_t)a.S) return;
    const TH *h = static_cast<const TH *>(a.h) + row * a.ldh;
    float x[NV][V], f[EARLY ? NV : 1][V];
#pragma unroll
    for (int u = 0; u < NV; u++) {
        const int j = tid + u * nt;
#pragma unroll
        for (int i = 0; i < V; i++) x[u][i] = 0.f;
        if (j < nvec) load_row<TH, V>(h + j * V, x[u]);
    }
    const auto fetch = [&](float (&to)[V], const float *from, int j) { if (j < nvec) load_row<float, V>(from + j * V, to); };
    if constexpr (SUM) {
        const TY *y = static_cast<const TY *>(a.y) + row * a.ldy;
        float p[NV][V], pf[EARLY ? NV : 1][V];
#pragma unroll
        for (int u = 0; u < NV; u++) {
            const int j = tid + u * nt;
#pragma unroll
            for (int i = 0; i < V; i++) p[u][i] = 0.f;
            if (j < nvec) load_row<TY, V>(y + j * V, p[u]);
        }
        if constexpr (EARLY) {
#pragma unroll
            for (int u = 0; u < NV; u++) {
                if (takes_weight(a.post)) fetch(pf[u], a.pw, tid + u * nt);
                if (takes_weight(a.variant)) fetch(f[u], a.w, tid + u * nt);
            }
        }
        float r = 1.f;
        if (a.post != W4A8_NORM_NONE) {
            double ss = 0.0;
#pragma unroll
            for (int u = 0; u < NV; u++) ss = squares(p[u], ss);
            r = (float)rsqrt(fma(cta_sum<WARP>(ss, sh_y), a.inv_k, a.eps));
        }
#pragma unroll
        for (int u = 0; u < NV; u++) {
            const int j = tid + u * nt;
            if (j < nvec) {
                if (a.post != W4A8_NORM_NONE) {
                    if (!EARLY && takes_weight(a.post)) fetch(pf[0], a.pw, j);
                    normed(p[u], r, pf[EARLY ? u : 0], a.post);
                }
                if (a.gate) {
                    float g[V];
                    load_row<float, V>(a.gate + row * a.ldg + j * V, g);
#pragma unroll
                    for (int i = 0; i < V; i++) p[u][i] = __fmul_rn(p[u][i], g[i]);
                }
#pragma unroll
                for (int i = 0; i < V; i++) x[u][i] = __fadd_rn(x[u][i], __fmul_rn(p[u][i], a.alpha));
            }
        }
    } else if constexpr (EARLY) {
#pragma unroll
        for (int u = 0; u < NV; u++)
            if (takes_weight(a.variant)) fetch(f[u], a.w, tid + u * nt);
    }
    if (a.h_out) {
        TH *o = static_cast<TH *>(a.h_out) + row * a.ldo;
#pragma unroll
        for (int u = 0; u < NV; u++) {
            const int j = tid + u * nt;
            if (j < nvec) store_row<TH, V>(o + j * V, x[u]);
        }
    }
    if (!a.n_out && !a.xq) return;
    if (a.variant != W4A8_NORM_NONE) {
        double ss = 0.0;
#pragma unroll
        for (int u = 0; u < NV; u++) ss = squares(x[u], ss);
        const float r = (float)rsqrt(fma(cta_sum<WARP>(ss, sh_h), a.inv_k, a.eps));
#pragma unroll
        for (int u = 0; u < NV; u++) {
            const int j = tid + u * nt;
            if (j < nvec) {
                if (!EARLY && takes_weight(a.variant)) fetch(f[0], a.w, j);
                normed(x[u], r, f[EARLY ? u : 0], a.variant);
            }
        }
    }
    if (a.n_out) {
        TH *o = static_cast<TH *>(a.n_out) + row * a.ldn;
#pragma unroll
        for (int u = 0; u < NV; u++) {
            const int j = tid + u * nt;
            if (j < nvec) store_row<TH, V>(o + j * V, x[u]);
        }
    }
    if (!a.xq) return;
    float amax[NV], top = 0.f;
#pragma unroll
    for (int u = 0; u < NV; u++) {
        amax[u] = 0.f;
#pragma unroll
        for (int i = 0; i < V; i++) amax[u] = fmaxf(amax[u], fabsf(x[u][i]));
        top = fmaxf(top, amax[u]);
    }
    if (a.group == 0) top = cta_max<WARP>(top, sh_max);
#pragma unroll
    for (int u = 0; u < NV; u++) {
        const int j = tid + u * nt;
        float m = top;
        if (a.group != 0) {                                            // the 32 / V lanes of a block: all of them have elements, or none
            m = amax[u];
#pragma unroll
            for (int o = 1; o < 32 / V; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        }
        const float d = quant_scale(m);
        uint32_t q[V / 4];
        int sum = 0;
#pragma unroll
        for (int c = 0; c < V / 4; c++) {
            int s4 = 0;
            q[c] = m != 0.f ? quantize4_pack(make_float4(x[u][4 * c], x[u][4 * c + 1], x[u][4 * c + 2], x[u][4 * c + 3]), d, s4) : 0u;
            sum += s4;
        }
        if (a.group != 0 && a.xsum) {
#pragma unroll
            for (int o = 1; o < 32 / V; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        }
        if (j < nvec) {
            int8_t *dst = a.xq + row * a.K + j * V;
            if constexpr (V == 4) *reinterpret_cast<uint32_t *>(dst) = q[0];
            else *reinterpret_cast<uint2 *>(dst) = make_uint2(q[0], q[1]);
            if (a.group != 0) {
                if (j % (32 / V) == 0) {
                    const size_t b = row * (a.K / 32) + j / (32 / V);
                    a.xs[b] = d;
                    if (a.xsum) a.xsum[b] = sum;
                }
            } else if (j == 0) {
                a.xs[row] = d;
            }
        }
    }
}

template <typename TH, typename TY, int EP, int MAXT, bool EARLY, bool SUM, bool WARP = false>
inline int launch_ep(Args a, int S, cudaStream_t st) {
    constexpr int WARP_ROWS = 4;
    a.S = S;
    const int need = (a.K + EP - 1) / EP;
    const dim3 grid(WARP ? (unsigned)(((long)S + WARP_ROWS - 1) / WARP_ROWS) : (unsigned)S), block(WARP ? WARP_ROWS * 32 : (need + 31) / 32 * 32);
    const cudaError_t e = launch_pdl(add_norm_kernel<TH, TY, EP, MAXT, EARLY, SUM, WARP>, grid, block, 0, st, a);
    if (e != cudaSuccess) return cuda_fail(e, "add_norm launch");
    return launch_status("add_norm");
}
template <typename TH, typename TY, bool SUM>
inline int launch_t(const Args &a, int S, cudaStream_t st) {
    if (a.K <= 32 * 16 && S > 4 * sm_count()) return launch_ep<TH, TY, 16, 128, false, SUM, true>(a, S, st);
    if constexpr (!SUM)
        if (a.K <= 32 * 32 && S > 4 * sm_count()) return launch_ep<TH, TY, 32, 128, false, SUM, true>(a, S, st);
    // Eight elements a thread while all rows run at once (some 56 registers a thread with a sum, 32 without), sixteen where they come in waves: us, sixteen / eight, norms of
    // 150 x 3840 3.7 / 3.0, 300 x 1024 3.1 / 2.2, 500 x 2048 3.9 / 3.1, but 300 x 5120 5.0 / 6.4; quantizers 200 x 5120 2.7 / 2.5, 590 x 4096 4.2 / 3.2.
    const int threads = (a.K / 8 + 31) / 32 * 32, at_once = (SUM ? 1152 : 2048) / threads;
    if (a.K <= 1024 * 8 && S <= sm_count() * (at_once < 1 ? 1 : at_once)) return launch_ep<TH, TY, 8, 1024, true, SUM>(a, S, st);
    if (a.K <= 512 * 16) return launch_ep<TH, TY, 16, 512, false, SUM>(a, S, st);
    if (a.K <= 1024 * 16) return launch_ep<TH, TY, 16, 1024, false, SUM>(a, S, st);
    return launch_ep<TH, TY, 32, 1024, false, SUM>(a, S, st);
}
template <typename TH>
inline int launch_y(const Args &a, int S, int dtype, int y_dtype, cudaStream_t st) {
    if (!a.y) return launch_t<TH, TH, false>(a, S, st);
    return y_dtype == dtype ? launch_t<TH, TH, true>(a, S, st) : launch_t<TH, float, true>(a, S, st);
}
inline int launch(const Args &a, int S, int dtype, int y_dtype, cudaStream_t st) {
    if (dtype == W4A8_F32) return launch_y<float>(a, S, dtype, W4A8_F32, st);
    return dtype == W4A8_F16 ? launch_y<__half>(a, S, dtype, y_dtype, st) : launch_y<__nv_bfloat16>(a, S, dtype, y_dtype, st);
}

}  // namespace addnorm
}  // namespace w4a8
