// 8-bit product with one scale for each row and each output channel, on the 5th-generation tensor cores:
//   Y[m][n] = float(sum_k xq[m][k] * wq[n][k]) * xs[m] * ws[n] + bias[n]
// The scales stand outside the sum, so the tensor core accumulates over all of K in int32 (exact: |sum| <= 131040 * 127^2 < 2^31) and the
// operands go from HBM to the MMA untouched: TMA brings both, 128 bytes of K at a time, in the swizzle that tcgen05.mma reads.
//
// The weights are the MMA's M side (128 channels, one to a TMEM lane), the rows of activations its N side: BT of them, any multiple of 16 up to
// 256, chosen on the host.  A step of one token then pads 16 columns and not 128 rows, and the epilogue's lanes hold neighbouring channels:
// what a warp stores of a row is contiguous.
//
// One CTA per SM, warp-specialised: warp 0 starts copies, warp 1 the MMAs, warps 2 to 5 convert, scale and store one tile while the next one
// accumulates in the other half of TMEM.  Where there are fewer tiles than SMs, the CTAs of a cluster share a tile's K (`split` of them), send
// their int32 sums to the CTA that owns the columns through distributed shared memory, and that one adds them: no workspace, no second
// launch, and the same bits, since integers add in any order.
#pragma once
#include <cuda.h>
#include "common.cuh"
#include "ptx_sm100.cuh"
#include "rows.cuh"
#include "tmap_cache.cuh"

namespace w4a8 {
namespace w8a8 {

constexpr int MAX_K = 131040;
constexpr int BW = 128, KT = 128;              // channels of a tile; bytes of K in a stage
constexpr int A_STAGE = BW * KT;
constexpr int MAX_STAGES = 12, EPI_WARPS = 4, THREADS = (2 + EPI_WARPS) * 32;
constexpr int SMEM_MAX = 227 * 1024, SMEM_FIXED = 1024 /* alignment */ + 512 /* barriers */;
constexpr int SPLIT_MAX = 8, SPLIT_BT = 64;    // CTAs that share a tile, and the widest tile that they share
enum : unsigned { ERR_PRODUCER = 0xA10u, ERR_MMA = 0xA20u, ERR_EPILOGUE = 0xA30u };

struct Args {
    const float *xs, *ws, *bias;
    void *y;
    int64_t ldy;
    int M, N, K, bt, stages, split, t_tiles, tiles, tmem_cols;
};

// The slot of a ring, and how often it came round.
struct Turn {
    int slot = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void next(int depth) {
        if (++slot == depth) { slot = 0; phase ^= 1u; }
    }
};

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t remote(uint32_t smem, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem), "r"(rank));
    return r;
}
__device__ __forceinline__ void st_remote(uint32_t addr, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }

__device__ __forceinline__ void prefetch_l2_2d(const void *tmap, int x, int y) {
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(tmap), "r"(x), "r"(y) : "memory");
}

__device__ __forceinline__ float scaled(int acc, float x, float w, float b) { return __fadd_rn(__fmul_rn(__fmul_rn(__int2float_rn(acc), x), w), b); }
__device__ __forceinline__ void put(float *p, float v) { *p = v; }
__device__ __forceinline__ void put(__half *p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void put(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }

template <typename T, bool SPLIT>
__global__ void __launch_bounds__(THREADS, 1) gemm_w8a8_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const Args a) {
    extern __shared__ unsigned char smem_dyn[];
    const uint32_t raw = ptx::smem_u32(smem_dyn), base = (raw + 1023u) & ~1023u;
    const uint32_t stage_bytes = A_STAGE + (uint32_t)a.bt * KT;
    const uint32_t bars = base + (uint32_t)a.stages * stage_bytes, recv = bars + 512;
    const auto FULL = [&](int s) { return bars + 8u * s; };
    const auto EMPTY = [&](int s) { return bars + 8u * (MAX_STAGES + s); };
    const auto T_FULL = [&](int s) { return bars + 8u * (2 * MAX_STAGES + s); };
    const auto T_EMPTY = [&](int s) { return bars + 8u * (2 * MAX_STAGES + 2 + s); };
    const uint32_t slot_addr = bars + 8u * (2 * MAX_STAGES + 4);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = SPLIT ? blockIdx.x % a.split : 0;
    const int nkt = (a.K + KT - 1) / KT;
    const int k_lo = SPLIT ? (int)((long)nkt * rank / a.split) : 0, k_hi = SPLIT ? (int)((long)nkt * (rank + 1) / a.split) : nkt;
    const int first = SPLIT ? blockIdx.x / a.split : blockIdx.x, step = SPLIT ? a.tiles : gridDim.x;

    if (threadIdx.x == 0) {
        for (int i = 0; i < a.stages; i++) { ptx::mbar_init(FULL(i), 1); ptx::mbar_init(EMPTY(i), 1); }
        for (int i = 0; i < 2; i++) { ptx::mbar_init(T_FULL(i), 1); ptx::mbar_init(T_EMPTY(i), EPI_WARPS); }
        ptx::mbar_fence_init();
        ptx::tma_prefetch_desc(&tmW);
        ptx::tma_prefetch_desc(&tmX);
    }
    if (warp == 1) {
        ptx::tmem_alloc(slot_addr, a.tmem_cols);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    if constexpr (SPLIT) cluster_sync();           // sums are sent to CTAs that have begun
    ptx::tc_fence_after_sync();
    uint32_t tmem;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(slot_addr));

    if (warp == 0) {
        if (lane == 0) {
            Turn ring;
            bool ok = true;
            // while the kernel in front drains, the first stages' weights are brought to L2: whatever it writes, L2 has it
            const int early = min(a.stages, k_hi - k_lo);
            for (int i = 0; i < early; i++) prefetch_l2_2d(&tmW, (k_lo + i) * KT, first / a.t_tiles * BW);
            pdl_wait();
            pdl_launch_dependents();
            for (int tile = first; tile < a.tiles && ok; tile += step)
                for (int kt = k_lo; kt < k_hi; kt++) {
                    if (!ptx::mbar_wait(EMPTY(ring.slot), ring.phase ^ 1u)) { dev_set_error(ERR_PRODUCER); ok = false; break; }
                    const uint32_t at = base + ring.slot * stage_bytes;
                    ptx::mbar_arrive_expect_tx(FULL(ring.slot), stage_bytes);
                    ptx::tma_load_2d(at, &tmW, kt * KT, tile / a.t_tiles * BW, FULL(ring.slot));
                    ptx::tma_load_2d(at + A_STAGE, &tmX, kt * KT, tile % a.t_tiles * a.bt, FULL(ring.slot));
                    ring.next(a.stages);
                }
            if (!ok) {                             // copies in flight land before the CTA's shared memory goes away
                const long long t0 = clock64();
                while (clock64() - t0 < (1ll << 21)) { }
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            pdl_wait();                            // before the first bounded wait: the kernel in front may take longer than any of them
            Turn ring, buf;
            const uint32_t idesc = ptx::umma_idesc_s8(BW, a.bt);
            bool ok = true;
            for (int tile = first; tile < a.tiles && ok; tile += step) {
                if (!ptx::mbar_wait(T_EMPTY(buf.slot), buf.phase ^ 1u)) { dev_set_error(ERR_MMA | 1); ok = false; break; }
                ptx::tc_fence_after_sync();
                for (int kt = k_lo; kt < k_hi; kt++) {
                    if (!ptx::mbar_wait(FULL(ring.slot), ring.phase)) { dev_set_error(ERR_MMA | 2); ok = false; break; }
                    ptx::tc_fence_after_sync();
                    const uint64_t w = ptx::umma_desc_k_sw128(base + ring.slot * stage_bytes), x = ptx::umma_desc_k_sw128(base + ring.slot * stage_bytes + A_STAGE);
                    const int parts = min(KT, a.K - kt * KT) / 32;
                    for (int p = 0; p < parts; p++) ptx::umma_i8(tmem + buf.slot * (a.tmem_cols / 2), w + 2 * p, x + 2 * p, idesc, kt > k_lo || p > 0);
                    ptx::umma_commit(EMPTY(ring.slot));
                    ring.next(a.stages);
                }
                if (ok) ptx::umma_commit(T_FULL(buf.slot));
                buf.next(2);
            }
            if (!ok) {                             // products in flight end before TMEM is given back
                const long long t0 = clock64();
                while (clock64() - t0 < (1ll << 21)) { }
            }
        }
    } else {
        pdl_wait();
        const int quad = warp & 3;                 // TMEM lanes [32 * quad, 32 * quad + 32) are this warp's
        Turn buf;
        for (int tile = first; tile < a.tiles; tile += step) {
            const int t0 = tile % a.t_tiles * a.bt, n = tile / a.t_tiles * BW + quad * 32 + lane, cols = min(a.bt, a.M - t0);
            const bool live = n < a.N;
            const float w = live ? a.ws[n] : 0.f, b = live && a.bias ? a.bias[n] : 0.f;
            T *y = static_cast<T *>(a.y) + (size_t)t0 * a.ldy + n;
            if (!ptx::mbar_wait_warp(T_FULL(buf.slot), buf.phase)) { dev_set_error(ERR_EPILOGUE); break; }
            ptx::tc_fence_after_sync();
            const uint32_t acc = tmem + ((uint32_t)(quad * 32) << 16) + buf.slot * (a.tmem_cols / 2);
            for (int c0 = 0; c0 < cols; c0 += 16) {
                uint32_t d[16];
                ptx::tmem_ld(acc + c0, d);
                ptx::tmem_ld_wait();
                if constexpr (SPLIT) {
                    const int own = (a.bt + a.split - 1) / a.split;    // columns [r * own, (r + 1) * own) are the r-th CTA's
#pragma unroll
                    for (int j = 0; j < 16; j++) {
                        const int c = c0 + j, r = c / own;
                        if (c < cols) st_remote(remote(recv + 4u * (((uint32_t)(rank * own + c - r * own) * BW) + quad * 32 + lane), r), d[j]);
                    }
                } else {
                    const float xv = c0 + lane < cols ? a.xs[t0 + c0 + lane] : 0.f;
#pragma unroll
                    for (int j = 0; j < 16; j++) {
                        const float v = scaled((int)d[j], __shfl_sync(0xffffffffu, xv, j), w, b);
                        if (live && c0 + j < cols) put(y + (size_t)(c0 + j) * a.ldy, v);
                    }
                }
            }
            ptx::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(T_EMPTY(buf.slot));
            buf.next(2);
        }
    }
    if constexpr (SPLIT) {
        __syncwarp();
        cluster_sync();                            // every sum has arrived; and nobody leaves while another one's are on their way
        if (warp >= 2) {
            const int quad = warp & 3, t0 = first % a.t_tiles * a.bt, n = first / a.t_tiles * BW + quad * 32 + lane, cols = min(a.bt, a.M - t0);
            const int own = (a.bt + a.split - 1) / a.split, c_hi = min(cols, (rank + 1) * own);
            const bool live = n < a.N;
            const float w = live ? a.ws[n] : 0.f, b = live && a.bias ? a.bias[n] : 0.f;
            T *y = static_cast<T *>(a.y) + (size_t)t0 * a.ldy + n;
            for (int c = rank * own; c < c_hi; c++) {
                int sum = 0;
                for (int r = 0; r < a.split; r++) {
                    int v;
                    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(recv + 4u * (((uint32_t)(r * own + c - rank * own) * BW) + quad * 32 + lane)));
                    sum += v;
                }
                const float v = scaled(sum, a.xs[t0 + c], w, b);
                if (live) put(y + (size_t)c * a.ldy, v);
            }
        }
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        __syncwarp();
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc(tmem, a.tmem_cols);
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------------------------
struct Plan { int bt, split; };
inline int ceil_div(long a, long b) { return (int)((a + b - 1) / b); }

inline Plan plan_for(int M, int N, int K, int sms) {
    const int w_tiles = ceil_div(N, BW), nkt = ceil_div(K, KT);
    if (M <= SPLIT_BT) {
        int split = sms / w_tiles;
        split = split < 1 ? 1 : split > SPLIT_MAX ? SPLIT_MAX : split;
        while (split > 1 && nkt / split < 4) split--;
        return {ceil_div(M, 16) * 16, split};
    }
    Plan best = {256, 1};
    double least = 1e30;
    for (int bt = 64; bt <= 256; bt += 16) {
        const long tiles = (long)w_tiles * ceil_div(M, bt);
        const double cost = (double)ceil_div(tiles, sms) * (bt < 128 ? 128 : bt);
        if (cost <= least) { least = cost; best.bt = bt; }
    }
    return best;
}

template <typename T, bool SPLIT>
inline int launch_t(Args a, const CUtensorMap &tmW, const CUtensorMap &tmX, cudaStream_t st) {
    auto kern = gemm_w8a8_kernel<T, SPLIT>;
    static PerDevice<bool> configured_dev;
    bool &configured = configured_dev.get();
    if (!configured) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MAX);
        if (e != cudaSuccess) return cuda_fail(e, "gemm_w8a8 smem opt-in");
        configured = true;
    }
    const int own = ceil_div(a.bt, a.split), recv = SPLIT ? a.split * own * BW * 4 : 0;
    const int stage = A_STAGE + a.bt * KT;
    int stages = (SMEM_MAX - SMEM_FIXED - recv) / stage;
    a.stages = stages > MAX_STAGES ? MAX_STAGES : stages;
    const int smem = a.stages * stage + SMEM_FIXED + recv, sms = sm_count();
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(SPLIT ? a.tiles * a.split : (a.tiles < sms ? a.tiles : sms));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (SPLIT) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = a.split; attr[n].val.clusterDim.y = 1; attr[n].val.clusterDim.z = 1;
        n++;
    }
    if (pdl_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        n++;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, tmW, tmX, a);
    if (e != cudaSuccess) return cuda_fail(e, "gemm_w8a8 launch");
    return launch_status("gemm_w8a8");
}

inline int launch(const int8_t *xq, const int8_t *wq, Args a, Plan p, int dtype, cudaStream_t st) {
    a.bt = p.bt;
    a.split = p.split;
    a.t_tiles = ceil_div(a.M, p.bt);
    const long tiles = (long)a.t_tiles * ceil_div(a.N, BW);
    if (tiles > 0x3fffffff) return fail(W4A8_ERR_UNSUPPORTED, "gemm_w8a8: %d x %d outputs", a.M, a.N);
    a.tiles = (int)tiles;
    a.tmem_cols = 32;
    while (a.tmem_cols < 2 * a.bt) a.tmem_cols *= 2;
    CUtensorMap tmW, tmX;
    int rc = tmap_cached(&tmW, wq, (uint64_t)a.K, (uint64_t)a.N, KT, BW, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B);
    if (rc != W4A8_OK) return rc;
    rc = tmap_cached(&tmX, xq, (uint64_t)a.K, (uint64_t)a.M, KT, (uint32_t)a.bt, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B);
    if (rc != W4A8_OK) return rc;
    const auto by_split = [&](auto t) {
        return p.split > 1 ? launch_t<decltype(t), true>(a, tmW, tmX, st) : launch_t<decltype(t), false>(a, tmW, tmX, st);
    };
    if (dtype == W4A8_F32) return by_split(float());
    return dtype == W4A8_F16 ? by_split(__half()) : by_split(__nv_bfloat16());
}

}  // namespace w8a8
}  // namespace w4a8
