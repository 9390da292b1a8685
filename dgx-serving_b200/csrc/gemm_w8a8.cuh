// 8-bit product with one scale for each row and each output channel, on the 5th-generation tensor cores:
//   Y[m][n] = float(sum_k xq[m][k] * wq[n][k]) * xs[m] * ws[n] + bias[n]
// The scales stand outside the sum, so the tensor core accumulates over all of K in int32 (exact: |sum| <= 131040 * 127^2 < 2^31) and the
// operands go from HBM to the MMA untouched: TMA brings both, 128 bytes of K at a time, in the swizzle that tcgen05.mma reads.
//
// The weights are the MMA's M side (128 channels, one to a TMEM lane), the rows of activations its N side: BT of them, any multiple of 16 up to
// 256, chosen on the host.  A step of one token then pads 16 columns and not 128 rows, and the epilogue's lanes hold neighbouring channels:
// what a warp stores of a row is contiguous.
//
// Large products run on pairs of CTAs (cta_group::2): 256 channels by bt rows, each CTA holding its 128 channels and half of the rows, one thread of the
// first CTA issuing the MMAs of both.  A byte in shared memory then serves twice the products: what fills shared memory bounds these products, and
// under the power cap what it costs to move.
//
// A row or two (ROWS) are quantized where they are used: every CTA takes the row's largest magnitude and writes its own part of K into the shared memory that the
// MMA reads, while the weights are on their way.  That saves the quantizer's launch, in which HBM is idle, and costs a read of the row from L2 for each SM
// (row_plan has what both take).
//
// One CTA per SM, warp-specialised: warp 0 starts copies, warp 1 the MMAs, warps 2 to 9 convert, scale and store one tile while the next one
// accumulates in the other half of TMEM.  Where there are fewer tiles than SMs, the CTAs of a cluster share a tile's K (`split` of them), send
// their int32 sums to the CTA that owns the columns through distributed shared memory, and that one adds them: no workspace, no second
// launch, and the same bits, since integers add in any order.
//
// Bounds and figures (us, in a graph): 2048 x 17408 x 5120 128 (2.85 POP/s; tensor pipe at three quarters, L2 at 44 %), 4096^3 52, 333 x 4091 x 3840 9.8 (676 KB of
// tiles into each of 128 CTAs, 5.4 at 64 bytes a cycle), 16 x 3840 x 15360 13.2 (4.5 TB/s; clusters' start and sums are 4 of it), 1 x 17408 x 5120 15.4 (5.8 TB/s).  The issuing warps stay converged and an elected
// lane issues: a lane that branches off alone took 300 cycles a K-tile for waits, descriptors and commits, and the first of these shapes 217 us.
#pragma once
#include <cuda.h>
#include "common.cuh"
#include "ptx_sm100.cuh"
#include "gemm_w8a8_plan.cuh"
#include "rows.cuh"
#include "tmap_cache.cuh"

namespace w4a8 {
namespace w8a8 {

enum : unsigned { ERR_PRODUCER = 0xA10u, ERR_MMA = 0xA20u, ERR_EPILOGUE = 0xA30u, ERR_SUMS = 0xA40u };

struct Args {
    const float *xs, *ws, *bias;
    void *y;
    int64_t ldy;
    int M, N, K, bw, bt, kp, stages, split, t_tiles, tiles, tmem_cols;
    const void *x;                             // ROWS: rows to quantize, their type, and where codes and scales go besides
    int64_t ldx;
    int8_t *xq_out;
    float *xs_out;
    int x_dtype;
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
// `bytes` of this CTA's shared memory to another one's of the cluster, where they count on an mbarrier.
__device__ __forceinline__ void send(uint32_t dst, uint32_t src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "r"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void epilogue_sync() { asm volatile("bar.sync 1, %0;" ::"n"(EPI_WARPS * 32) : "memory"); }

// ---- two CTAs of a cluster as a pair (cta_group::2): ranks 0 and 1 ---------------------------------------------------------------------
__device__ __forceinline__ void tmem_alloc_pair(uint32_t dst_smem, uint32_t columns) {          // a warp of each CTA
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst_smem), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t tmem, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns));
}
// Into this CTA's memory; the bytes count on an mbarrier of either CTA.
__device__ __forceinline__ void tma_load_2d_pair(uint32_t lead, uint32_t dst_smem, const void *tmap, int x, int y, uint32_t bar) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                 "@q cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n\t}"
                 ::"r"(dst_smem), "l"(tmap), "r"(x), "r"(y), "r"(bar), "r"(lead) : "memory");
}
__device__ __forceinline__ void umma_s8_pair(uint32_t lead, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                 "@q tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(lead) : "memory");
}
// Arrives on the barrier at this place in both CTAs.
__device__ __forceinline__ void umma_commit_pair(uint32_t lead, uint32_t bar) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t"
                 "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::"r"(bar), "h"((uint16_t)3), "r"(lead) : "memory");
}
__device__ __forceinline__ void arrive_remote(uint32_t bar) { asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }

__device__ __forceinline__ void prefetch_l2_2d(const void *tmap, int x, int y) {
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(tmap), "r"(x), "r"(y) : "memory");
}

__device__ __forceinline__ float scaled(int acc, float x, float w, float b) { return __fadd_rn(__fmul_rn(__fmul_rn(__int2float_rn(acc), x), w), b); }
__device__ __forceinline__ void put(float *p, float v) { *p = v; }
__device__ __forceinline__ void put(__half *p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void put(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }

// Eight elements of a row of any type.
__device__ __forceinline__ void load8(const void *row, int64_t at, int dtype, float (&v)[8]) {
    if (dtype == W4A8_F32) load_row<float, 8>(static_cast<const float *>(row) + at, v);
    else if (dtype == W4A8_F16) load_row<__half, 8>(static_cast<const __half *>(row) + at, v);
    else load_row<__nv_bfloat16, 8>(static_cast<const __nv_bfloat16 *>(row) + at, v);
}

enum Mode { ONE, SPLIT, PAIR };                // a tile is one CTA's; several share its K; two share its channels

template <typename T, Mode MODE, bool ROWS>
__global__ void __launch_bounds__(THREADS, 1) gemm_w8a8_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const Args a) {
    extern __shared__ unsigned char smem_dyn[];
    const uint32_t raw = ptx::smem_u32(smem_dyn), base = (raw + 1023u) & ~1023u;
    const uint32_t x_rows = MODE == PAIR ? a.bt / 2 : a.bt, part_bytes = A_STAGE + (ROWS ? 0 : x_rows * KT), stage_bytes = part_bytes * a.kp;
    const uint32_t bars = base + (uint32_t)a.stages * stage_bytes, recv = bars + 512, x_at = recv + (MODE == SPLIT ? (uint32_t)(a.split * ((a.bt + a.split - 1) / a.split) * LANES * 4) : 0u) + 512;   // (x_at: a multiple of 1024)
    const auto FULL = [&](int s) { return bars + 8u * s; };
    const auto EMPTY = [&](int s) { return bars + 8u * (MAX_STAGES + s); };
    const auto T_FULL = [&](int s) { return bars + 8u * (2 * MAX_STAGES + s); };
    const auto T_EMPTY = [&](int s) { return bars + 8u * (2 * MAX_STAGES + 2 + s); };
    const uint32_t sums_full = bars + 8u * (2 * MAX_STAGES + 4), slot_addr = bars + 8u * (2 * MAX_STAGES + 5), x_full = bars + 8u * (2 * MAX_STAGES + 6);
    float *row_max = reinterpret_cast<float *>(smem_dyn + (bars - raw) + 256), *row_scale = row_max + EPI_WARPS;       // ROWS
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = MODE == ONE ? 0 : blockIdx.x % a.split;   // in the cluster
    const int nkt = (a.K + KT - 1) / KT;
    const int k_lo = MODE == SPLIT ? (int)((long)nkt * rank / a.split) : 0, k_hi = MODE == SPLIT ? (int)((long)nkt * (rank + 1) / a.split) : nkt;
    const int first = MODE == ONE ? blockIdx.x : blockIdx.x / a.split, step = MODE == SPLIT ? a.tiles : MODE == PAIR ? gridDim.x / 2 : gridDim.x;
    const int my_row = MODE == PAIR ? rank * LANES : 0;        // this CTA's channels in a tile
    // SPLIT: rows [r * own, (r + 1) * own) of the tile are the r-th CTA's to finish
    const int own = MODE == SPLIT ? (a.bt + a.split - 1) / a.split : 0, tile_rows = min(a.bt, a.M - first % a.t_tiles * a.bt);
    const auto rows_of = [&](int r) { return max(0, min(own, tile_rows - r * own)); };

    if (threadIdx.x == 0) {
        for (int i = 0; i < a.stages; i++) { ptx::mbar_init(FULL(i), 1); ptx::mbar_init(EMPTY(i), 1); }
        for (int i = 0; i < 2; i++) { ptx::mbar_init(T_FULL(i), 1); ptx::mbar_init(T_EMPTY(i), MODE == PAIR ? 2 * EPI_WARPS : EPI_WARPS); }
        if constexpr (ROWS) ptx::mbar_init(x_full, EPI_WARPS * 32);
        if constexpr (MODE == SPLIT) {
            ptx::mbar_init(sums_full, 1);
            ptx::mbar_arrive_expect_tx(sums_full, (uint32_t)((a.split - 1) * rows_of(rank) * LANES * 4));
        }
        ptx::mbar_fence_init();
        ptx::tma_prefetch_desc(&tmW);
        ptx::tma_prefetch_desc(&tmX);
    }
    if (warp == 1) {
        if constexpr (MODE == PAIR) tmem_alloc_pair(slot_addr, a.tmem_cols);
        else {
            ptx::tmem_alloc(slot_addr, a.tmem_cols);
            ptx::tmem_relinquish();
        }
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    if constexpr (MODE != ONE) cluster_sync();                 // others' memory and barriers are used once they have begun
    ptx::tc_fence_after_sync();
    uint32_t tmem;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(slot_addr));

    if (warp == 0) {
        const uint32_t lead = ptx::elected();
        Turn ring;
        // while the kernel in front drains, the first stages' weights are brought to L2: whatever it writes, L2 has it
        const int early = min(a.stages * a.kp, k_hi - k_lo);
        if (lead)
            for (int i = 0; i < early; i++) prefetch_l2_2d(&tmW, (k_lo + i) * KT, first / a.t_tiles * a.bw + my_row);
        pdl_wait();
        pdl_launch_dependents();
        bool ok = true;
        for (int tile = first; tile < a.tiles && ok; tile += step) {
            const int w_row = tile / a.t_tiles * a.bw + my_row, x_row = tile % a.t_tiles * a.bt + (MODE == PAIR ? rank * x_rows : 0);
            for (int kt = k_lo; kt < k_hi; kt += a.kp) {
                if (!ptx::mbar_wait_warp(EMPTY(ring.slot), ring.phase ^ 1u)) { dev_set_error(ERR_PRODUCER); ok = false; break; }
                const int parts = min(a.kp, k_hi - kt);
                uint32_t at = base + ring.slot * stage_bytes;
                const uint32_t bar = MODE == PAIR ? remote(FULL(ring.slot), 0) : FULL(ring.slot);      // a pair's bytes count where its MMAs are issued
                if (MODE != PAIR || rank == 0) ptx::mbar_arrive_expect_tx(lead, FULL(ring.slot), (uint32_t)(a.bw + (ROWS ? 0 : a.bt)) * KT * parts);
                for (int p = 0; p < parts; p++, at += part_bytes) {
                    if constexpr (MODE == PAIR) {
                        tma_load_2d_pair(lead, at, &tmW, (kt + p) * KT, w_row, bar);
                        tma_load_2d_pair(lead, at + A_STAGE, &tmX, (kt + p) * KT, x_row, bar);
                    } else {
                        ptx::tma_load_2d(lead, at, &tmW, (kt + p) * KT, w_row, bar);
                        if constexpr (!ROWS) ptx::tma_load_2d(lead, at + A_STAGE, &tmX, (kt + p) * KT, x_row, bar);
                    }
                }
                ring.next(a.stages);
            }
        }
        if (!ok) {                                             // copies in flight land before the CTA's shared memory goes away
            const long long t0 = clock64();
            while (clock64() - t0 < (1ll << 21)) { }
        }
    } else if (warp == 1 && rank != 0 && MODE == PAIR) {
        pdl_wait();                                            // the first CTA issues for both
    } else if (warp == 1) {
        pdl_wait();                                            // before the first bounded wait: the kernel in front may take longer than any of them
        const uint32_t lead = ptx::elected(), idesc = ptx::umma_idesc_s8(MODE == PAIR ? 2 * LANES : LANES, a.bt);
        Turn ring, buf;
        bool ok = true;
        if (ROWS && !ptx::mbar_wait_warp(x_full, 0)) { dev_set_error(ERR_MMA | 3); ok = false; }
        for (int tile = first; tile < a.tiles && ok; tile += step) {
            if (!ptx::mbar_wait_warp(T_EMPTY(buf.slot), buf.phase ^ 1u)) { dev_set_error(ERR_MMA | 1); ok = false; break; }
            ptx::tc_fence_after_sync();
            const uint32_t acc = tmem + buf.slot * (a.tmem_cols / 2);
            for (int kt = k_lo; kt < k_hi; kt += a.kp) {
                if (!ptx::mbar_wait_warp(FULL(ring.slot), ring.phase)) { dev_set_error(ERR_MMA | 2); ok = false; break; }
                ptx::tc_fence_after_sync();
                uint32_t at = base + ring.slot * stage_bytes;
                for (int q = kt; q < min(kt + a.kp, k_hi); q++, at += part_bytes) {
                    const uint64_t w = ptx::umma_desc_k_sw128(at), x = ptx::umma_desc_k_sw128(ROWS ? x_at + (uint32_t)(q - k_lo) * a.bt * KT : at + A_STAGE);
                    const int parts = min(KT, a.K - q * KT) / 32;
#pragma unroll
                    for (int p = 0; p < KT / 32; p++)
                        if (p < parts) {
                            if constexpr (MODE == PAIR) umma_s8_pair(lead, acc, w + 2 * p, x + 2 * p, idesc, q > k_lo || p > 0);
                            else ptx::umma_s8(lead, acc, w + 2 * p, x + 2 * p, idesc, q > k_lo || p > 0);
                        }
                }
                if constexpr (MODE == PAIR) umma_commit_pair(lead, EMPTY(ring.slot));
                else ptx::umma_commit(lead, EMPTY(ring.slot));
                ring.next(a.stages);
            }
            if (ok) {
                if constexpr (MODE == PAIR) umma_commit_pair(lead, T_FULL(buf.slot));
                else ptx::umma_commit(lead, T_FULL(buf.slot));
            }
            buf.next(2);
        }
        if (!ok) {                                             // products in flight end before TMEM is given back
            const long long t0 = clock64();
            while (clock64() - t0 < (1ll << 21)) { }
        }
    } else {
        pdl_wait();
        // TMEM lanes [32 * quad, 32 * quad + 32) are this warp's, and of their columns every second 32
        const int quad = warp & 3, row = quad * 32 + lane, side = (warp - 2) >> 2;
        Turn buf;
        if constexpr (ROWS) {
            const int t = threadIdx.x - 64, vectors = a.K / 8;
            const bool keep = first == 0;                      // the first tile's CTAs also store what the caller gets
            constexpr int KEPT = 4, TURN = EPI_WARPS * 32;     // vectors of eight that a thread keeps between the two passes, all loaded at once
            const int lo = k_lo * (KT / 8), hi = min(k_hi * (KT / 8), vectors);
            for (int m = 0; m < a.M; m++) {
                const char *src = static_cast<const char *>(a.x) + (size_t)m * a.ldx * (a.x_dtype == W4A8_F32 ? 4 : 2);
                float kept[KEPT][8], top = 0.f;
#pragma unroll
                for (int u = 0; u < KEPT; u++) {
#pragma unroll
                    for (int i = 0; i < 8; i++) kept[u][i] = 0.f;
                    if (t + u * TURN < vectors) load8(src, 8 * (t + u * TURN), a.x_dtype, kept[u]);
                }
                const auto largest = [&](const float (&v)[8]) {
#pragma unroll
                    for (int i = 0; i < 8; i++) top = fmaxf(top, fabsf(v[i]));
                };
#pragma unroll
                for (int u = 0; u < KEPT; u++) largest(kept[u]);
                for (int j = t + KEPT * TURN; j < vectors; j += TURN) {
                    float v[8];
                    load8(src, 8 * j, a.x_dtype, v);
                    largest(v);
                }
                top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
                if (lane == 0) row_max[warp - 2] = top;
                epilogue_sync();
#pragma unroll
                for (int i = 0; i < EPI_WARPS; i++) top = fmaxf(top, row_max[i]);
                const float d = quant_scale(top);
                if (t == 0) {
                    row_scale[m] = d;
                    if (keep && rank == 0) a.xs_out[m] = d;
                }
                const auto codes = [&](int j, const float (&v)[8]) {
                    if (j < lo || j >= hi) return;
                    int sum;
                    uint32_t q0 = 0, q1 = 0;
                    if (top != 0.f) {
                        q0 = quantize4_pack(make_float4(v[0], v[1], v[2], v[3]), d, sum);
                        q1 = quantize4_pack(make_float4(v[4], v[5], v[6], v[7]), d, sum);
                    }
                    const int kt = j / (KT / 8) - k_lo, chunk = j % (KT / 8) / 2;          // m < 8: rows of one group of eight, swizzled by their number
                    asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(x_at + (uint32_t)kt * a.bt * KT + m * KT + ((chunk ^ m) << 4) + (j & 1) * 8), "r"(q0), "r"(q1) : "memory");
                    if (keep) *reinterpret_cast<uint2 *>(a.xq_out + (size_t)m * a.K + 8 * j) = make_uint2(q0, q1);
                };
#pragma unroll
                for (int u = 0; u < KEPT; u++) codes(t + u * TURN, kept[u]);
                for (int j = t + KEPT * TURN; j < hi; j += TURN) {
                    float v[8];
                    load8(src, 8 * j, a.x_dtype, v);
                    codes(j, v);
                }
                epilogue_sync();                               // row_max is read, row_scale is there
            }
            ptx::fence_proxy_async_smem();
            ptx::mbar_arrive(x_full);
        }
        for (int tile = first; tile < a.tiles; tile += step) {
            // what the outputs need besides the sums, while these are on their way: lane l has the scales of rows l, l + 32, ... of its columns
            const int n = tile / a.t_tiles * a.bw + my_row + row, t0 = tile % a.t_tiles * a.bt + (MODE == SPLIT ? rank * own : 0), rows = MODE == SPLIT ? rows_of(rank) : min(a.bt, a.M - t0);
            const bool live = my_row + row < a.bw && n < a.N;
            constexpr int XR = MODE == SPLIT ? SPLIT_BT / 2 / 64 : 4;
            float x[XR];
#pragma unroll
            for (int i = 0; i < XR; i++) {
                const int c = MODE == SPLIT ? 2 * (32 * i + lane) + side : 64 * i + 32 * side + lane;
                x[i] = c < rows ? (ROWS ? row_scale[t0 + c] : a.xs[t0 + c]) : 0.f;
            }
            const float w = live ? a.ws[n] : 0.f, b = live && a.bias ? a.bias[n] : 0.f;
            T *y = static_cast<T *>(a.y) + (size_t)t0 * a.ldy + n;
            bool ok = ptx::mbar_wait_warp(T_FULL(buf.slot), buf.phase);
            if (!ok) dev_set_error(ERR_EPILOGUE);
            if (MODE != SPLIT && !ok) break;               // (SPLIT: its warps meet below, whatever each one's wait came to)
            ptx::tc_fence_after_sync();
            const uint32_t acc = tmem + ((uint32_t)(quad * 32) << 16) + buf.slot * (a.tmem_cols / 2);
            const int columns = MODE == SPLIT ? tile_rows : rows;
#pragma unroll
            for (int i = 0; i < (MODE == SPLIT ? SPLIT_BT / 64 : 4); i++) {
                const int c0 = 64 * i + 32 * side;
                if (c0 >= columns) break;
                uint32_t d[32];
                if (c0 + 16 < a.bt) ptx::tmem_ld(acc + c0, d);
                else {                                         // an odd number of sixteens: the last one alone
                    uint32_t half[16];
                    ptx::tmem_ld(acc + c0, half);
#pragma unroll
                    for (int j = 0; j < 16; j++) d[j] = half[j];
                }
                ptx::tmem_ld_wait();
                T *p = y + (size_t)c0 * a.ldy;
#pragma unroll
                for (int j = 0; j < 32; j++) {
                    if constexpr (MODE == SPLIT) {             // every product has been read: the stages' memory is free
                        if (c0 + j < columns) asm volatile("st.shared.u32 [%0], %1;" ::"r"(base + 4u * ((c0 + j) * LANES + row)), "r"(d[j]) : "memory");
                    } else {
                        const float v = scaled((int)d[j], __shfl_sync(0xffffffffu, x[i], j), w, b);
                        if (live && c0 + j < columns) put(p, v);
                        p += a.ldy;
                    }
                }
            }
            if constexpr (MODE == SPLIT) {
                ptx::fence_proxy_async_smem();
                epilogue_sync();
                if (warp == 2 && lane < a.split && lane != rank && rows_of(lane) > 0)
                    send(remote(recv + (uint32_t)(rank * own * LANES * 4), lane), base + (uint32_t)(lane * own * LANES * 4), (uint32_t)(rows_of(lane) * LANES * 4), remote(sums_full, lane));
                if (!ptx::mbar_wait_warp(sums_full, 0)) { dev_set_error(ERR_SUMS); ok = false; }
                if (!ok) {                                     // sums on their way land before the cluster's memory goes away
                    const long long since = clock64();
                    while (clock64() - since < (1ll << 21)) { }
                    break;
                }
                static_assert(XR == 1);
                const int *mine = reinterpret_cast<const int *>(smem_dyn + (base - raw)) + row, *theirs = reinterpret_cast<const int *>(smem_dyn + (recv - raw)) + row;
                for (int j = 0; 2 * j + side < rows; j += 4) {             // every second row, four of them at a time
                    int sum[4] = {};
                    for (int r = 0; r < a.split; r++) {
                        const int *from = (r == rank ? mine : theirs) + (r * own + 2 * j + side) * LANES;
#pragma unroll
                        for (int q = 0; q < 4; q++)
                            if (2 * (j + q) + side < rows) sum[q] += from[2 * q * LANES];
                    }
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        const int c = 2 * (j + q) + side;
                        const float v = scaled(sum[q], __shfl_sync(0xffffffffu, x[0], j + q), w, b);
                        if (live && c < rows) put(y + (size_t)c * a.ldy, v);
                    }
                }
            }
            ptx::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                if constexpr (MODE == PAIR) arrive_remote(remote(T_EMPTY(buf.slot), 0));
                else ptx::mbar_arrive(T_EMPTY(buf.slot));
            }
            buf.next(2);
        }
    }
    if constexpr (MODE != ONE) {                               // nobody leaves while another CTA reads or writes its memory
        __syncwarp();
        cluster_sync();
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        __syncwarp();
        ptx::tc_fence_after_sync();
        if constexpr (MODE == PAIR) tmem_dealloc_pair(tmem, a.tmem_cols);
        else ptx::tmem_dealloc(tmem, a.tmem_cols);
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------------------------
template <typename T, Mode MODE, bool ROWS = false>
inline int opt_in() {                                                  // a per-device function attribute
    static PerDevice<bool> configured_dev;
    bool &configured = configured_dev.get();
    if (!configured) {
        const cudaError_t e = cudaFuncSetAttribute(gemm_w8a8_kernel<T, MODE, ROWS>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MAX);
        if (e != cudaSuccess) return cuda_fail(e, "gemm_w8a8 smem opt-in");
        configured = true;
    }
    return W4A8_OK;
}

// How many clusters fit depends on how the GPU's SMs are grouped: asked of the driver once a device.
inline int caps_of(Caps *out) {
    static PerDevice<Caps> caps_dev;
    Caps &caps = caps_dev.get();
    if (caps.sms == 0) {
        Caps c = {};
        int rc = opt_in<float, SPLIT>();
        if (rc != W4A8_OK) return rc;
        for (int n = 2; n <= SPLIT_MAX; n++) {
            cudaLaunchConfig_t cfg = {};
            cudaLaunchAttribute attr;
            attr.id = cudaLaunchAttributeClusterDimension;
            attr.val.clusterDim.x = n; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
            cfg.gridDim = dim3(n); cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = SMEM_MAX; cfg.attrs = &attr; cfg.numAttrs = 1;
            const cudaError_t e = cudaOccupancyMaxActiveClusters(&c.clusters[n], gemm_w8a8_kernel<float, SPLIT, false>, &cfg);
            if (e != cudaSuccess) return cuda_fail(e, "gemm_w8a8 clusters");
        }
        c.sms = sm_count();
        caps = c;
    }
    *out = caps;
    return W4A8_OK;
}
// The plan of a shape, kept for the shapes called last (a decode loop has a few; finding one takes some microseconds).
inline int plan_cached(int M, int N, int K, Plan *out) {
    struct Slot { int M, N, K, dev; Plan plan; };
    static Slot slots[PLAN_SLOTS] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) dev = 0;
    Slot &s = slots[plan_slot(M, N, K, dev)];
    if (s.M != M || s.N != N || s.K != K || s.dev != dev) {
        Caps caps;
        const int rc = caps_of(&caps);
        if (rc != W4A8_OK) return rc;
        s = {M, N, K, dev, plan_for(M, N, K, caps)};
    }
    *out = s.plan;
    return W4A8_OK;
}

template <typename T, Mode MODE, bool ROWS>
inline int launch_t(Args a, const Plan &p, const CUtensorMap &tmW, const CUtensorMap &tmX, cudaStream_t st) {
    auto kern = gemm_w8a8_kernel<T, MODE, ROWS>;
    const int rc = opt_in<T, MODE, ROWS>();
    if (rc != W4A8_OK) return rc;
    a.stages = ROWS ? row_stages_for(p, a.K) : stages_for(p);
    const int smem = ROWS ? row_smem_for(p, a.K) : smem_for(p), sms = sm_count();
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(MODE == SPLIT ? a.tiles * a.split : MODE == PAIR ? 2 * (a.tiles < p.at_once ? a.tiles : p.at_once) : (a.tiles < sms ? a.tiles : sms));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (MODE != ONE) {
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
    a.bw = p.bw;
    a.bt = p.bt;
    a.kp = p.kp;
    a.split = p.pair ? 2 : p.split;                // CTAs of a cluster
    a.t_tiles = ceil_div(a.M, p.bt);
    const long tiles = (long)a.t_tiles * ceil_div(a.N, p.bw);
    if (tiles > 0x3fffffff) return fail(W4A8_ERR_UNSUPPORTED, "gemm_w8a8: %d x %d outputs", a.M, a.N);
    a.tiles = (int)tiles;
    a.tmem_cols = 32;
    while (a.tmem_cols < (p.split > 1 ? 1 : 2) * a.bt) a.tmem_cols *= 2;
    CUtensorMap tmW, tmX;
    int rc = tmap_cached(&tmW, wq, (uint64_t)a.K, (uint64_t)a.N, KT, (uint32_t)(p.pair ? LANES : a.bw), CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
    if (rc != W4A8_OK) return rc;
    rc = tmap_cached(&tmX, xq, (uint64_t)a.K, (uint64_t)a.M, KT, (uint32_t)(p.pair ? a.bt / 2 : a.bt), CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B);
    if (rc != W4A8_OK) return rc;
    const auto by_split = [&](auto t) {
        using O = decltype(t);
        if (a.x) return p.split > 1 ? launch_t<O, SPLIT, true>(a, p, tmW, tmX, st) : launch_t<O, ONE, true>(a, p, tmW, tmX, st);
        if (p.pair) return launch_t<O, PAIR, false>(a, p, tmW, tmX, st);
        return p.split > 1 ? launch_t<O, SPLIT, false>(a, p, tmW, tmX, st) : launch_t<O, ONE, false>(a, p, tmW, tmX, st);
    };
    if (dtype == W4A8_F32) return by_split(float());
    return dtype == W4A8_F16 ? by_split(__half()) : by_split(__nv_bfloat16());
}

}  // namespace w8a8
}  // namespace w4a8
