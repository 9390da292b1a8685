// The 8-bit paged KV cache: block tables and slot maps from request lengths, rows into the blocks, rows out of them.
//
// Cache layout: codes k, v [num_blocks][heads][block][dim] int8 and scales [num_blocks][heads] fp32; a token's element is code * scale.
// A block holds `block` consecutive tokens of one request; slot = block id * block + token's place in it.
#pragma once
#include "common.cuh"
#include "rows.cuh"

namespace w4a8 {
namespace kv {

using w4a8::Row;

constexpr int LONGEST = 0x7fffffff - 511;     // tokens of a request: positions a few tiles on are counted in 31 bits too
enum { ERR_BLOCK_ID = 0x900u, ERR_SLOT = 0x901u, ERR_LENGTH = 0x902u };   // codes of the device-side error word

// ---- block tables and slot maps ----------------------------------------------------------------------------------------------------
// One launch.  Every CTA scans all requests (two sums at once, in the halves of a 64-bit number: new tokens and fresh blocks before each
// request; R numbers from L2 cost less than a second launch that would hand the sums over) and then fills its share of the slots and
// of the fresh table entries, finding the request of each by bisection of the sums in shared memory.
constexpr int PLAN_THREADS = 512;
constexpr int PLAN_MAX_R = 16384;

struct PlanArgs {
    const int32_t *kv_len, *new_len, *free_blocks, *first;
    int32_t *table, *seq_len, *cu_new, *slot, *position, *status;
    int R, block, width, num_free, T;
    unsigned last_id;                          // the largest id that slots can be made of
};

__device__ __forceinline__ int ceil_div64(long long a, int b) { return (int)((a + b - 1) / b); }

// Largest i in [0, n) with cum[i] <= x (cum ascending, cum[0] = 0 <= x).
__device__ __forceinline__ int last_at_most(const int *cum, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (cum[mid] <= x) lo = mid; else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(PLAN_THREADS) kv_plan_kernel(PlanArgs a) {
    extern __shared__ int plan_smem[];
    int *cu = plan_smem, *before = plan_smem + a.R + 1;          // new tokens, fresh blocks in front of request i
    __shared__ unsigned long long part[PLAN_THREADS / 32 + 1];
    __shared__ int totals[4];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_wait();
    pdl_launch_dependents();
    if (tid < 4) totals[tid] = 0;
    const int first = max(0, min(a.first[0], a.num_free)), avail = a.num_free - first;
    unsigned long long carry = 0;
    for (int base = 0; base < a.R; base += PLAN_THREADS) {
        const int r = base + tid;
        unsigned long long v = 0;
        if (r < a.R) {
            const int kv = max(0, a.kv_len[r]), nw = max(0, a.new_len[r]);
            const int want = ceil_div64((long long)kv + nw, a.block);
            const int need = want <= a.width && (long long)kv + nw <= LONGEST ? want - ceil_div64(kv, a.block) : 0;
            v = ((unsigned long long)(unsigned)nw << 32) | (unsigned)need;
        }
        unsigned long long s = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long u = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += u;
        }
        if (lane == 31) part[warp] = s;
        __syncthreads();
        if (warp == 0) {
            unsigned long long w = lane < PLAN_THREADS / 32 ? part[lane] : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned long long u = __shfl_up_sync(0xffffffffu, w, o);
                if (lane >= o) w += u;
            }
            if (lane < PLAN_THREADS / 32) part[lane] = w;
        }
        __syncthreads();
        const unsigned long long excl = carry + (warp ? part[warp - 1] : 0) + s - v;
        if (r < a.R) { cu[r] = (int)(excl >> 32); before[r] = (int)(unsigned)excl; }
        carry += part[PLAN_THREADS / 32 - 1];
        __syncthreads();
    }
    if (tid == 0) { cu[a.R] = (int)(carry >> 32); before[a.R] = (int)(unsigned)carry; }
    __syncthreads();

    // served: the request's tokens fit its table row, and it needs no block or the free list reaches for it and all in front of it
    const auto served = [&](int r, int kv) {
        const int want = ceil_div64((long long)kv + (cu[r + 1] - cu[r]), a.block);
        return want <= a.width && (long long)kv + (cu[r + 1] - cu[r]) <= LONGEST && (before[r + 1] == before[r] || before[r + 1] <= avail);
    };
    const int gt = blockIdx.x * PLAN_THREADS + tid, gn = gridDim.x * PLAN_THREADS;
    if (blockIdx.x == 0) {
        int taken_to = 0, unserved = 0, tokens = 0;
        for (int r = tid; r < a.R; r += PLAN_THREADS) {
            const int kv = max(0, a.kv_len[r]), nw = cu[r + 1] - cu[r];
            const bool ok = served(r, kv);
            a.seq_len[r] = ok ? kv + nw : 0;
            a.cu_new[r] = cu[r];
            if (ok) { tokens += nw; if (before[r + 1] > before[r]) taken_to = max(taken_to, before[r + 1]); }
            else unserved++;
        }
        if (taken_to) atomicMax(&totals[0], taken_to);
        if (unserved) atomicAdd(&totals[1], unserved);
        if (tokens) atomicAdd(&totals[2], tokens);
        __syncthreads();
        if (tid == 0) {
            a.cu_new[a.R] = cu[a.R];
            a.status[0] = first + totals[0];
            a.status[1] = totals[1];
            a.status[2] = totals[0];
            a.status[3] = totals[2];
        }
    }
    bool bad = false;
    for (int t = gt; t < a.T; t += gn) {
        int slot = -1, pos = -1;
        if (t < cu[a.R]) {
            const int r = last_at_most(cu, a.R, t), kv = max(0, a.kv_len[r]);
            if (served(r, kv)) {
                pos = kv + t - cu[r];
                const int b = pos / a.block, have = ceil_div64(kv, a.block);
                const int id = b < have ? a.table[(size_t)r * a.width + b] : a.free_blocks[first + before[r] + b - have];
                // no slot can be made of any id (its product may wrap to a slot of another request)
                const bool good = (unsigned)id <= a.last_id;
                slot = good ? id * a.block + pos % a.block : -1;
                bad = bad || !good;
            }
        }
        a.slot[t] = slot;
        if (a.position) a.position[t] = pos;
    }
    if (bad) dev_set_error(ERR_BLOCK_ID);
    for (int f = gt; f < before[a.R] && f < avail; f += gn) {
        const int r = last_at_most(before, a.R, f), kv = max(0, a.kv_len[r]);
        if (served(r, kv)) a.table[(size_t)r * a.width + ceil_div64(kv, a.block) + f - before[r]] = a.free_blocks[first + f];
    }
}

// ---- rows into the blocks -----------------------------------------------------------------------------------------------------------
// A group is the run of consecutive rows whose slots follow one another inside one block; a CTA takes the groups that begin among its
// `span` rows, and a team of TEAM threads one head of the keys or of the values.  The group's largest magnitude, with the scale of tokens that
// the block held before, gives the block's new scale; codes that were there are rounded to it.  The rows are in registers between the two
// (HOLD pieces of 16 bytes a thread), beyond that they are read again, from L1 or L2: the magnitude is needed before the first code.
// A warp is the team while a block's rows fit its registers: all loads are in flight at once and no barrier is needed.  8192 rows of 8 heads of
// 128 in bf16, keys and values (33 MB read, 17 written): 13.7 us, 34 with teams of 128 threads, a walk row by row and divisions in place.
constexpr int APPEND_THREADS = 128;
constexpr int APPEND_SPAN = 128;              // a CTA looks at span + block rows' slots at most
constexpr int APPEND_HOLD = 8;

struct AppendArgs {
    const void *k, *v;
    const int32_t *slot;
    int8_t *kc, *vc;
    float *ks, *vs;
    long long ldk;
    int T, heads, block, span;
    int slots;                                // num_blocks * block
};

// Four codes by the reciprocal r of the scale, and whether they are certainly those of the division: m holds the integer nearest to x * r in its low
// byte, t is the distance to it; x * r is within 127 * 2^-23 of x / scale, so only a distance near a half can round otherwise.  (r 0: zeros.)
__device__ __forceinline__ uint32_t quantize4_fast(float4 v, float r, bool &sure) {
    constexpr float MAGIC = 12582912.0f, TIE = 0.5f - 0x1p-15f;
    const float m0 = fmaf(v.x, r, MAGIC), m1 = fmaf(v.y, r, MAGIC), m2 = fmaf(v.z, r, MAGIC), m3 = fmaf(v.w, r, MAGIC);
    const float t0 = fmaf(v.x, r, MAGIC - m0), t1 = fmaf(v.y, r, MAGIC - m1), t2 = fmaf(v.z, r, MAGIC - m2), t3 = fmaf(v.w, r, MAGIC - m3);
    sure = sure && fabsf(t0) <= TIE && fabsf(t1) <= TIE && fabsf(t2) <= TIE && fabsf(t3) <= TIE;
    return __byte_perm(__byte_perm(__float_as_uint(m0), __float_as_uint(m1), 0x0040), __byte_perm(__float_as_uint(m2), __float_as_uint(m3), 0x0040), 0x5410);
}

template <typename T, int D, int TEAM>
__global__ void __launch_bounds__(APPEND_THREADS, 8) kv_append_q8_kernel(AppendArgs a) {
    constexpr int N = Row<T>::N, VPR = D / N, NW = APPEND_THREADS / 32, HOLD = TEAM == 32 ? APPEND_HOLD : 2;
    __shared__ uint32_t follow[(2 * APPEND_SPAN + 32) / 32];      // bit i: row t0 + i continues the group of the row before it
    __shared__ float red[NW];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, me = tid % TEAM;
    const int u = blockIdx.y * (APPEND_THREADS / TEAM) + tid / TEAM, h = u >> 1, t0 = blockIdx.x * a.span;
    const bool values = u & 1;
    const T *src = static_cast<const T *>(values ? a.v : a.k) + (size_t)h * D;
    int8_t *codes = values ? a.vc : a.kc;
    float *scales = values ? a.vs : a.ks;
    pdl_wait();
    pdl_launch_dependents();
    const int look = min(a.T - t0, a.span + a.block);
    for (int i = tid; i < ((look + 31) & ~31); i += APPEND_THREADS) {
        const int t = t0 + i;
        bool f = false;
        if (i < look && t > 0) {
            const int s = a.slot[t], before = a.slot[t - 1];
            f = s > 0 && s < a.slots && (s & (a.block - 1)) != 0 && before == s - 1;
        }
        const uint32_t bits = __ballot_sync(0xffffffffu, f);
        if (lane == 0) follow[i >> 5] = bits;
    }
    __syncthreads();
    if (h >= a.heads) return;                                      // a whole team; only teams of a warp have such
    const auto head = [&](int i) {                                 // the first row from i on that begins a group, or `look`
        for (; i < look; i = (i | 31) + 1) {
            const uint32_t w = ~follow[i >> 5] >> (i & 31);
            if (w) return min(look, i + __ffs((int)w) - 1);
        }
        return look;
    };
    const int bshift = 31 - __clz(a.block);
    int next;
    for (int i0 = head(0); i0 < a.span && t0 + i0 < a.T; i0 = next) {
        next = head(i0 + 1);                                       // a group ends inside its block: slot % block == 0 does not follow
        const int slot = a.slot[t0 + i0];
        if (slot < 0) continue;                                    // a padded row
        if (slot >= a.slots) { if (me == 0) dev_set_error(ERR_SLOT); continue; }
        const int m = next - i0, b = slot >> bshift, off = slot & (a.block - 1);
        const size_t unit = (size_t)b * a.heads + h;
        int8_t *dst = codes + (unit * a.block + off) * D;
        const T *rows = src + (size_t)(t0 + i0) * a.ldk;
        const int nvec = m * VPR;
        const float was = off > 0 ? scales[unit] : 0.f;
        uint4 hold[HOLD];
        float amax = 0.f;
#pragma unroll
        for (int j = 0; j < HOLD; j++) {
            const int e = me + j * TEAM;
            hold[j] = e < nvec ? *reinterpret_cast<const uint4 *>(rows + (size_t)(e / VPR) * a.ldk + (e % VPR) * N) : make_uint4(0, 0, 0, 0);
        }
        const auto widest = [&](uint4 raw) {
            float x[N];
            Row<T>::unpack(raw, x);
#pragma unroll
            for (int q = 0; q < N; q++) amax = fmaxf(amax, fabsf(x[q]));
        };
#pragma unroll
        for (int j = 0; j < HOLD; j++) widest(hold[j]);
#pragma unroll 4
        for (int e = me + HOLD * TEAM; e < nvec; e += TEAM)
            widest(*reinterpret_cast<const uint4 *>(rows + (size_t)(e / VPR) * a.ldk + (e % VPR) * N));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        if constexpr (TEAM > 32) {
            __syncthreads();                                       // red of the group before has been read
            if (lane == 0) red[warp] = amax;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < NW; w++) amax = fmaxf(amax, red[w]);
        }
        const float now = fmaxf(was, quant_scale(amax));
#pragma unroll
        for (int j = 0; j < HOLD; j++)                             // unpacked anew below: kept as floats they would be twice the registers
            asm volatile("" : "+r"(hold[j].x), "+r"(hold[j].y), "+r"(hold[j].z), "+r"(hold[j].w));
        // q = rint(x / now) by the reciprocal; a piece in which that is not sure to round alike is left for the divisions below, so that these are in
        // the code once (inlined, or called from each place, they took the registers of two thirds of the warps)
        float r = 0.f;
        if (now > 0.f) asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(now));
        const bool in_range = now == 0.f || (now >= 0x1p-100f && now <= 0x1p100f);
        unsigned long long unsure = 0;                             // pieces of this thread, at most 128 rows * 64 pieces / 128 threads of them
        const auto keep = [&](int e, const uint32_t (&w)[N / 4]) {
            uint32_t *out = reinterpret_cast<uint32_t *>(dst + (size_t)e * N);       // the group's rows are one piece of memory
            if constexpr (N == 4) out[0] = w[0];
            else *reinterpret_cast<uint2 *>(out) = make_uint2(w[0], w[1]);
        };
        const auto put = [&](int j, uint4 raw) {
            float x[N];
            Row<T>::unpack(raw, x);
            uint32_t w[N / 4];
            bool sure = in_range;
#pragma unroll
            for (int q = 0; q < N / 4; q++) w[q] = quantize4_fast(make_float4(x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]), r, sure);
            keep(me + j * TEAM, w);
            if (!sure) unsure |= 1ull << j;
        };
#pragma unroll
        for (int j = 0; j < HOLD; j++)
            if (me + j * TEAM < nvec) put(j, hold[j]);
#pragma unroll 1
        for (int j = HOLD, e = me + HOLD * TEAM; e < nvec; j++, e += TEAM)
            put(j, *reinterpret_cast<const uint4 *>(rows + (size_t)(e / VPR) * a.ldk + (e % VPR) * N));
        for (; unsure; unsure &= unsure - 1) {
            const int e = me + (__ffsll((long long)unsure) - 1) * TEAM;
            float x[N];
            Row<T>::unpack(*reinterpret_cast<const uint4 *>(rows + (size_t)(e / VPR) * a.ldk + (e % VPR) * N), x);
            uint32_t w[N / 4];
#pragma unroll
            for (int q = 0; q < N / 4; q++) w[q] = quantize4_div(make_float4(x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]), now);
            keep(e, w);
        }
        if (off > 0 && now > was) {                                // the codes in front, to the new scale
            const float ratio = __fdiv_rn(was, now);
            uint32_t *old = reinterpret_cast<uint32_t *>(codes + unit * a.block * D);
            for (int e = me; e < off * (D / 4); e += TEAM) {
                const uint32_t w = old[e];
                uint32_t r = 0;
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const float x = __fmul_rn((float)(int8_t)(w >> (8 * q)), ratio);
                    r |= ((uint32_t)(__float2int_rn(x)) & 0xFFu) << (8 * q);
                }
                old[e] = r;
            }
        }
        if constexpr (TEAM == 32) __syncwarp();                    // everybody has read `was` (teams of several warps: before the last barrier)
        if (me == 0) scales[unit] = now;
    }
}

// ---- rows out of the blocks ---------------------------------------------------------------------------------------------------------
constexpr int READ_THREADS = 256;

struct ReadArgs {
    const int8_t *kc, *vc;
    const float *ks, *vs;
    const int32_t *table, *begin, *cu;
    void *k, *v;
    long long ldo;
    int R, T, width, heads, block, num_blocks, tokens;       // tokens: per CTA, at most READ_THREADS
};

template <typename T, int D>
__global__ void __launch_bounds__(READ_THREADS) kv_read_q8_kernel(ReadArgs a) {
    constexpr int N = Row<T>::N, VPR = D / N;
    __shared__ int unit[READ_THREADS], place[READ_THREADS];
    const int tid = threadIdx.x, t0 = blockIdx.x * a.tokens;
    pdl_wait();
    pdl_launch_dependents();
    // the request of the CTA's first token: the sums are tested in READ_THREADS places at a time
    int lo = 0, hi = a.R;
    const int end = a.cu[a.R];
    while (hi - lo > 1) {
        const int step = (hi - lo + READ_THREADS - 1) / READ_THREADS, at = lo + tid * step;
        const int past = __syncthreads_count(at < hi && (tid == 0 || a.cu[at] <= t0));
        lo += (past - 1) * step;
        hi = min(hi, lo + step);
    }
    if (tid < a.tokens) {
        int id = -1, off = 0;
        const int t = t0 + tid;
        if (t < a.T && t < end) {
            while (lo + 1 < a.R && a.cu[lo + 1] <= t) lo++;
            const long long pos = (long long)a.begin[lo] + t - a.cu[lo];
            const long long b = pos / a.block;
            if (pos >= 0 && b < a.width) {
                id = a.table[(size_t)lo * a.width + b];
                off = (int)(pos - b * a.block);
            }
            if (id < 0 || id >= a.num_blocks) { dev_set_error(ERR_BLOCK_ID); id = -1; }
        }
        unit[tid] = id;
        place[tid] = off;
    }
    __syncthreads();
    const int8_t *codes = blockIdx.y ? a.vc : a.kc;
    const float *scales = blockIdx.y ? a.vs : a.ks;
    T *out = static_cast<T *>(blockIdx.y ? a.v : a.k);
    // piece c of token i, without a division for each; codes to fp32 through the bits of 2^23 + code + 128 (8192 tokens of 8 heads of 128, keys and
    // values, to bf16: 9.7 us, 10.1 with a conversion each and divisions; the bytes alone take 7.7)
    const int per = a.heads * VPR, total = a.tokens * per, step_i = READ_THREADS / per, step_c = READ_THREADS - step_i * per;
    int i = tid / per, c = tid - i * per;
#pragma unroll 4
    for (int e = tid; e < total; e += READ_THREADS) {
        const int at = unit[i];
        if (at >= 0) {
            const int h = c / VPR, x = (c - h * VPR) * N;
            const size_t u = (size_t)at * a.heads + h;
            const int8_t *p = codes + (u * a.block + place[i]) * D + x;
            const float s = scales[u];
            uint32_t w[N / 4];
            if constexpr (N == 4) w[0] = *reinterpret_cast<const uint32_t *>(p);
            else {
                const uint2 v = *reinterpret_cast<const uint2 *>(p);
                w[0] = v.x;
                w[1] = v.y;
            }
            float y[N];
#pragma unroll
            for (int q = 0; q < N / 4; q++)
#pragma unroll
                for (int j = 0; j < 4; j++) y[4 * q + j] = (__uint_as_float(__byte_perm(w[q] ^ 0x80808080u, 0x4B000000u, 0x7540 + j)) - 8388736.f) * s;
            *reinterpret_cast<uint4 *>(out + (size_t)(t0 + i) * a.ldo + h * D + x) = Row<T>::pack(y);
        }
        i += step_i;
        c += step_c;
        if (c >= per) { c -= per; i++; }
    }
}

// ---- launches -----------------------------------------------------------------------------------------------------------------------
inline int launch_plan(const PlanArgs &a, cudaStream_t st) {
    const size_t smem = (size_t)(a.R + 1) * 2 * sizeof(int);
    // what a launch gets without asking, 48 KB, has to hold the kernel's own arrays too: asked for once, for the most requests
    static PerDevice<bool> configured;
    if (!configured.get()) {
        cudaError_t e = cudaFuncSetAttribute(kv_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (PLAN_MAX_R + 1) * 2 * (int)sizeof(int));
        if (e != cudaSuccess) return cuda_fail(e, "kv_plan smem opt-in");
        configured.get() = true;
    }
    const int want = (a.T + 4 * PLAN_THREADS - 1) / (4 * PLAN_THREADS), most = sm_count();
    const int grid = want < 1 ? 1 : (want < most ? want : most);
    cudaError_t e = launch_pdl(kv_plan_kernel, dim3(grid), dim3(PLAN_THREADS), smem, st, a);
    return e == cudaSuccess ? launch_status("kv_plan") : cuda_fail(e, "kv_plan launch");
}

// Rows per CTA: few enough that the CTAs fill the GPU, a block's worth at most (then about every CTA has one group).
inline int append_span(int T, int heads, int block) {
    const long most = (long)sm_count() * 16;
    long span = ((long)T * heads * 2 + most - 1) / most;
    return (int)(span < 1 ? 1 : (span > block ? block : span));
}
// Tokens per CTA of the read: about four of a thread's pieces each, fewer where that leaves SMs idle.
inline int read_tokens(int T, int heads, int dim) {
    long n = (long)READ_THREADS * 4 * 8 / ((long)heads * dim);
    const long fill = ((long)T * 2 + sm_count() * 4 - 1) / (sm_count() * 4);
    if (n > fill) n = fill;
    return (int)(n < 1 ? 1 : (n > READ_THREADS ? READ_THREADS : n));
}

template <typename T, int D>
inline int launch_append_t(const AppendArgs &a, cudaStream_t st) {
    const bool warps = a.block * (D / Row<T>::N) <= 32 * APPEND_HOLD;          // a warp holds a block's rows
    const int units = 2 * a.heads, teams = warps ? APPEND_THREADS / 32 : 1;
    const dim3 grid((a.T + a.span - 1) / a.span, (units + teams - 1) / teams);
    cudaError_t e = warps ? launch_pdl(kv_append_q8_kernel<T, D, 32>, grid, dim3(APPEND_THREADS), 0, st, a)
                          : launch_pdl(kv_append_q8_kernel<T, D, APPEND_THREADS>, grid, dim3(APPEND_THREADS), 0, st, a);
    return e == cudaSuccess ? launch_status("kv_append_q8") : cuda_fail(e, "kv_append_q8 launch");
}
template <typename T, int D>
inline int launch_read_t(const ReadArgs &a, cudaStream_t st) {
    const dim3 grid((a.T + a.tokens - 1) / a.tokens, 2);
    cudaError_t e = launch_pdl(kv_read_q8_kernel<T, D>, grid, dim3(READ_THREADS), 0, st, a);
    return e == cudaSuccess ? launch_status("kv_read_q8") : cuda_fail(e, "kv_read_q8 launch");
}

// The kernel of an element type and a head size: fn(T(), integral_constant D).
template <typename Fn>
inline int by_type(int dtype, int dim, Fn &&fn) {
    const auto with = [&](auto t) {
        if (dim == 64) return fn(t, std::integral_constant<int, 64>());
        if (dim == 128) return fn(t, std::integral_constant<int, 128>());
        return fn(t, std::integral_constant<int, 256>());
    };
    if (dtype == W4A8_F32) return with(float());
    if (dtype == W4A8_F16) return with(__half());
    return with(__nv_bfloat16());
}

}  // namespace kv
}  // namespace w4a8
