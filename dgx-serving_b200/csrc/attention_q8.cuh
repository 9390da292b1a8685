// Attention of a few queries a request over the 8-bit paged KV cache: a stream of the blocks through shared memory.
//
//   s[i,j] = scale * ks[block(j)] * sum_d q[i,d] K[j,d]           (K, V: the int8 codes)
//   o[i]   = sum_j exp(s[i,j] - m) vs[block(j)] V[j] / sum_j exp(s[i,j] - m),   j over what query i sees
//
// What bounds it: the codes have to come from HBM once, 2 * dim bytes a token and kv head.  Everything else is arranged not to be in the way:
//  - Work is cut evenly: the (request, kv head, row group) pairs' key tiles of 64 tokens, laid one behind the other, are divided into equal
//    ranges, one per resident CTA, whatever the lengths.  A pair that several CTAs share leaves partial results (sum, maximum, weighted
//    values) in the workspace; the last of them to finish joins them in the order of the ranges, so the result does not depend on who is
//    last.  One launch.
//  - One warp brings the tiles by TMA into a ring (128-byte swizzle), following the block table; a block never has to be a whole tile.
//  - Four warps take 16 keys of a tile each and keep their own running maximum, sum and weighted values in registers for all rows (queries
//    x heads of the group); they meet once at the end of a pair.
//  - Q K^T: the codes enter mma.sync m16n8k32 (s8, int32 sums, exact) as they lie in memory.  A query row is cut into three signed digits of base
//    128 relative to its largest magnitude (2^-22 of it); digits one and two lie in rows g and g + 8 of one instruction, the third of rows g and
//    g + 8 in another.  fp16 operands need five instructions to widen four codes: decode of 64 requests 148 us.
//  - P V: mma.sync m16n8k16 with fp16 operands and fp32 sums, since the weights need a floating point; codes are exact in fp16 (one permute
//    and one packed subtraction for two of them).  The weight that enters is x = exp(s - B) * vs, in base 2 with the block's scale in the
//    exponent: one multiply-add and one exp2, the sum divides vs out again once per block.  B is the row's reference: the largest x was 2^8 when
//    it was chosen, and it moves, rescaling what is summed, only when an x would pass 2^15.  16-bit rows round x to fp16 once (2^-12, below the
//    rounding of a 16-bit result), fp32 rows take two terms (22 bits) in rows g and g + 8.
//    tcgen05 has nothing to add here: at most 32 rows meet each key, the instruction's 128 would be padding.
#pragma once
#include "kv_cache.cuh"
#include "ptx_sm100.cuh"
#include "tmap_cache.cuh"

namespace w4a8 {
namespace attn {

constexpr int TK = 64;                     // tokens of a tile
constexpr int CW = 4;                      // consumer warps: 16 tokens of the tile each
constexpr int THREADS = (CW + 1) * 32;
constexpr int MAX_R = 2048;                // requests of one launch (their sums lie in shared memory)
constexpr int FEW_ROWS = 64;                // rows (queries x heads of a group) of a request that the streaming kernel takes at most
constexpr int MIN_TILES = 2;               // a CTA takes at least so many tiles: joining costs about two tiles' time
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr unsigned ERR_WAIT = 0xA00u;

struct Args {
    const void *q;
    void *out;
    float *lse;
    const float *ks, *vs;
    const int32_t *table, *cu_q, *seq_len;
    long long ldq, ldo;
    int R, T, width, Hq, Hkv, G, block, num_blocks, stages;
    int causal, window;
    float scale, softcap;
    int few;                               // rows (queries * G) of a request that this kernel takes at most; more are another kernel's
    unsigned *count;                       // workspace: arrivals per CTA, zero between calls
    float2 *part_ml;                       // [2 * CTAs][rows] maximum, sum
    float *part;                           // [2 * CTAs][rows][dim]
};

__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint4 &a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_s8(int (&c)[4], const uint4 &a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
// Bytes (lo: 0 and 1, hi: 2 and 3) of a word of codes + 128 as two fp16 numbers, minus the 128 again: 0x6400 | u is 1024 + u.
template <int SEL>
__device__ __forceinline__ uint32_t codes_f16(uint32_t u) {
    const uint32_t w = __byte_perm(u, 0x64646464u, SEL);
    return h2_bits(__hsub2(*reinterpret_cast<const __half2 *>(&w), __half2half2(__ushort_as_half(0x6480))));   // 1152
}

// ---- which keys and how much work ----------------------------------------------------------------------------------------------------
struct Request {
    int q0, n, seq, lo, tiles, groups;       // first row of Q, rows, tokens, first token that any row sees, tiles from its tile on, row groups
};
__device__ __forceinline__ Request request(const Args &a, int r, int rows_per_group) {
    Request x;
    x.q0 = max(0, min(a.cu_q[r], a.T));
    x.n = max(0, min(a.cu_q[r + 1], a.T) - x.q0);
    x.seq = max(0, a.seq_len[r]);
    const long long most = (long long)a.width * a.block;
    if (x.seq > most) { x.seq = (int)most; dev_set_error(kv::ERR_LENGTH); }
    x.lo = a.window > 0 ? max(0, x.seq - x.n - a.window + 1) : 0;
    // at least one tile, so that rows that see nothing are written too
    x.tiles = x.seq > x.lo ? (x.seq + TK - 1) / TK - x.lo / TK : 1;
    const int rows = x.n * a.G;
    x.groups = rows <= a.few ? (rows + rows_per_group - 1) / rows_per_group : 0;
    return x;
}

// A CTA's range of units cut at the pairs' ends.
struct Segment {
    int r, h, rg, tile, tiles;               // tiles [tile, tile + tiles) of the pair's
    int pair0, pair_tiles;                   // the pair's first unit, its tiles
    Request x;
};
struct Walk {
    const Args &a;
    const unsigned *cum;
    unsigned u, end;
    int rpg;
    __device__ __forceinline__ Walk(const Args &a_, const unsigned *cum_, unsigned u0, unsigned u1, int rpg_) : a(a_), cum(cum_), u(u0), end(u1), rpg(rpg_), r(-1) {}
    int r;
    Request x;
    __device__ __forceinline__ bool next(Segment &s) {
        if (u >= end) return false;
        if (r < 0) {
            int lo = 0, hi = a.R;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (cum[mid] <= u) lo = mid; else hi = mid;
            }
            r = lo;
            x = request(a, r, rpg);
        } else if (u >= cum[r + 1]) {
            do r++; while (cum[r + 1] <= u);
            x = request(a, r, rpg);
        }
        const unsigned in = u - cum[r], pair = in / (unsigned)x.tiles, t = in - pair * (unsigned)x.tiles;
        s.r = r;
        s.h = (int)(pair % (unsigned)a.Hkv);
        s.rg = (int)(pair / (unsigned)a.Hkv);
        s.tile = (int)t;
        s.tiles = (int)min((unsigned)x.tiles - t, end - u);
        s.pair0 = (int)(u - t);
        s.pair_tiles = x.tiles;
        s.x = x;
        u += s.tiles;
        return true;
    }
};

// Where the tile's tokens go for the warps' reads to meet no bank twice (checked for each head size): a tile is planes of 128-byte rows, the
// 16-byte piece c of row r at c ^ (r & 7).  dim 128 and 256: a row is a token, a plane 128 elements.  dim 64: a row is two tokens.
template <int D> struct Tile {
    static constexpr int PLANES = D == 256 ? 2 : 1, ROW_TOKENS = D == 64 ? 2 : 1;
    static constexpr int PLANE_BYTES = TK * D / PLANES, BYTES = TK * D;
    // token of the instruction's column n (0..7) in the t-th (0, 1) group of eight: QK and PV agree on it
    static __device__ __forceinline__ int token(int t, int n) { return D == 64 ? 4 * (n >> 1) + (n & 1) + 2 * t : n + 8 * t; }
    // address of piece c (0..7 of a plane's 128 elements; 0..3 with dim 64) of token k
    static __device__ __forceinline__ uint32_t piece(int k, int c, int plane) {
        if constexpr (D == 64) { const int row = k >> 1; return row * 128 + ((((k & 1) * 4 + c) ^ (row & 7)) << 4); }
        else return plane * PLANE_BYTES + k * 128 + ((c ^ (k & 7)) << 4);
    }
    // dim of the first of the 16 elements that lane column c (0..3) reads in the p-th step of QK: piece and plane
    static constexpr int STEPS = D / 64;
    static __device__ __forceinline__ int qk_piece(int c, int p) { return D == 64 ? c : 2 * c + (p & 1); }
    static __device__ __forceinline__ int qk_plane(int p) { return p >> 1; }
};

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
    return v;
}
__device__ __forceinline__ float4 lds_f4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
    return v;
}

// Four consecutive elements of a row of Q as floats.
__device__ __forceinline__ float4 load4(const float *p) { return *reinterpret_cast<const float4 *>(p); }
__device__ __forceinline__ float4 load4(const __half *p) {
    const uint2 w = *reinterpret_cast<const uint2 *>(p);
    const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&w.x)), b = __half22float2(*reinterpret_cast<const __half2 *>(&w.y));
    return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ float4 load4(const __nv_bfloat16 *p) {
    const uint2 w = *reinterpret_cast<const uint2 *>(p);
    return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xFFFF0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xFFFF0000u));
}
__device__ __forceinline__ void store4(float *p, float4 v) { *reinterpret_cast<float4 *>(p) = v; }
__device__ __forceinline__ void store4(__half *p, float4 v) {
    *reinterpret_cast<uint2 *>(p) = make_uint2(h2_bits(__floats2half2_rn(v.x, v.y)), h2_bits(__floats2half2_rn(v.z, v.w)));
}
__device__ __forceinline__ void store4(__nv_bfloat16 *p, float4 v) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
}

// Power of two that brings a row whose largest magnitude is amax near 2^13, and its inverse times `scale`.
__device__ __forceinline__ float row_factor(float amax) {
    if (!(amax > 0.f) || !(amax < __int_as_float(0x7f800000))) return 1.f;
    int e = 13 - (((__float_as_int(amax) >> 23) & 0xFF) - 127);
    e = max(-126, min(126, e));
    return __int_as_float((e + 127) << 23);
}

constexpr int SLOT_SCALES = 4;              // blocks of a tile at most (blocks of 16 tokens)
constexpr size_t CONTROL = 1280;            // barriers and the stages' scales: ks, log2 vs, 1 / vs, vs == 0
__device__ __forceinline__ float lg2(float x) { float y; asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
// cap * tanh(x) * log2 e with x in units of cap: 1 - 2 / (1 + e^2x), whose error is that of a number near 1
__device__ __forceinline__ float capped(float x, float cap) { return cap * LOG2E * (1.f - __fdividef(2.f, 1.f + ex2(x * (2.f * LOG2E)))); }

// Digits of base 128 of four elements, as bytes of a word: v = d1 * 128^(n-1) + ..., |v| <= 127 * 128^(n-1); v becomes what is left.
__device__ __forceinline__ uint32_t digit4(float4 &v, float unit, float per) {
    const float a = rintf(v.x * per), b = rintf(v.y * per), c = rintf(v.z * per), d = rintf(v.w * per);
    v.x = fmaf(a, -unit, v.x); v.y = fmaf(b, -unit, v.y); v.z = fmaf(c, -unit, v.z); v.w = fmaf(d, -unit, v.w);
    const uint32_t lo = __byte_perm((uint32_t)(int)a, (uint32_t)(int)b, 0x0040), hi = __byte_perm((uint32_t)(int)c, (uint32_t)(int)d, 0x0040);
    return __byte_perm(lo, hi, 0x5410);
}

// Position of the f-th float4 of a row of `dim` floats in the buffer where the warps' results meet: no bank twice when the four lane columns
// write eight (dim 64: four) float4s each, side by side.
template <int D>
__device__ __forceinline__ int meet_pos(int f, int row) {
    if constexpr (D == 64) return (f & ~3) | ((f & 3) ^ (((f >> 3) & 1) + 2 * (row & 1)));
    else return (f & ~7) | ((f & 7) ^ (((f >> 3) & 3) + 4 * (row & 1)));
}

// R rows (queries x heads of a group) to a CTA's tile: 8, 16, 32.  A thread has rows g + 8 i.
template <typename T, int D, int R>
struct Shape {
    static constexpr bool SPLIT = std::is_same<T, float>::value;      // fp32 rows: two terms of the weights
    static constexpr int NR = R / 8, SETS = NR + (NR + 1) / 2, PM = SPLIT ? NR : (NR + 1) / 2;    // instructions' row tiles of QK and of PV
    static constexpr bool QREG = SETS * D / 8 <= 64;                  // the digits in registers
    static constexpr size_t MEET_BYTES = (size_t)CW * R * D * 4, Q_BYTES = QREG ? 0 : (size_t)SETS * (D / 32) * 32 * 16;
    static constexpr size_t STAGE_BYTES = 2 * (size_t)Tile<D>::BYTES;
    static constexpr size_t FIXED = 1280 + CONTROL + MEET_BYTES + Q_BYTES + (size_t)CW * R * 8 + R * 4;    // and 4 bytes a request
    // two CTAs an SM where each still has a ring of four stages and the weighted values fit the registers
    static constexpr int PER_SM = PM * D <= 128 && FIXED + 1024 + 4 * STAGE_BYTES <= 113 * 1024 ? 2 : 1;
    static inline size_t fixed_bytes(int n) { return FIXED + ((size_t)n + 4) * 4; }
    static inline int stages(int n) {
        const size_t k = ((PER_SM == 2 ? 113 : 226) * 1024 - fixed_bytes(n)) / STAGE_BYTES;
        return k < 12 ? (int)k : 12;
    }
};

template <typename T, int D, int R>
__global__ void __launch_bounds__(THREADS, Shape<T, D, R>::PER_SM) attention_q8_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Args a) {
    using S = Shape<T, D, R>;
    using L = Tile<D>;
    constexpr int NR = S::NR, SETS = S::SETS, PM = S::PM, ROWS = R, KS = D / 32, NT = D / 8;
    constexpr bool SPLIT = S::SPLIT, QREG = S::QREG;
    extern __shared__ unsigned char smem_raw[];
    // ring first (1024-byte aligned for the swizzle), then the rest
    unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char *ring = smem, *p = ring + (size_t)a.stages * S::STAGE_BYTES;
    unsigned char *control = p; p += CONTROL;
    float *meet = reinterpret_cast<float *>(p); p += S::MEET_BYTES;
    uint4 *qs = reinterpret_cast<uint4 *>(p); p += S::Q_BYTES;
    float2 *ml = reinterpret_cast<float2 *>(p); p += (size_t)CW * ROWS * 8;
    float *row_fac = reinterpret_cast<float *>(p); p += ROWS * 4;
    unsigned *cum = reinterpret_cast<unsigned *>(p);
    const uint32_t bar = ptx::smem_u32(control), scales_at = bar + 256, ring_at = ptx::smem_u32(ring);
    const auto FULL = [&](int s) { return bar + 8u * s; };
    const auto EMPTY = [&](int s) { return bar + 128u + 8u * s; };
    __shared__ unsigned wsum[THREADS / 32], last_flag;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        for (int s = 0; s < a.stages; s++) { ptx::mbar_init(FULL(s), 1); ptx::mbar_init(EMPTY(s), CW); }
        ptx::mbar_fence_init();
        ptx::tma_prefetch_desc(&map_k);
        ptx::tma_prefetch_desc(&map_v);
    }
    pdl_wait();
    pdl_launch_dependents();
    // units in front of each request
    unsigned carry = 0;
    for (int base = 0; base < a.R; base += THREADS) {
        const int r = base + tid;
        unsigned v = 0;
        if (r < a.R) { const Request x = request(a, r, ROWS); v = (unsigned)x.groups * (unsigned)a.Hkv * (unsigned)x.tiles; }
        unsigned s = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const unsigned t = __shfl_up_sync(0xffffffffu, s, o); if (lane >= o) s += t; }
        if (lane == 31) wsum[warp] = s;
        __syncthreads();
        unsigned in_front = carry;
        for (int w = 0; w < warp; w++) in_front += wsum[w];
        if (r < a.R) cum[r] = in_front + s - v;
        for (int w = 0; w < THREADS / 32; w++) carry += wsum[w];
        __syncthreads();
    }
    if (tid == 0) cum[a.R] = carry;
    __syncthreads();
    const unsigned U = carry;
    if (U == 0) return;
    // equal ranges for as many CTAs as get MIN_TILES each
    const unsigned P = min(gridDim.x, max(1u, U / MIN_TILES)), cta = blockIdx.x;
    if (cta >= P) return;
    const auto bound = [&](unsigned i) { return (unsigned)((unsigned long long)i * U / P); };
    const auto cta_of = [&](unsigned u) { return (unsigned)(((unsigned long long)(u + 1) * P - 1) / U); };
    const unsigned u0 = bound(cta), u1 = bound(cta + 1);
    const int bshift = 31 - __clz(a.block), piece_tokens = min(a.block, TK), pshift = 31 - __clz(piece_tokens), pieces = TK / piece_tokens;

    if (warp == CW) {
        // ---- producer: lane = one piece (the part of a block that lies in a tile); a batch is 32 pieces ------------------------------
        Walk walk(a, cum, u0, u1, ROWS);
        Segment s;
        int stage = 0, used = 0;                                   // used: stages filled so far (the ring's first round needs no wait)
        uint32_t phase = 0;
        bool more = walk.next(s), ok = true;
        int t_next = 0;                                            // next tile of the segment to look up
        const int per_batch = 32 / pieces;
        struct Batch { int tiles, row, tok; float ks, vs; bool mine; } b;
        int phys = 0;
        const auto look_up = [&]() {                               // the table entry of this lane's piece of the next batch
            b.tiles = 0; b.mine = false;
            if (!more) return;
            b.tiles = min(per_batch, s.tiles - t_next);
            const int t = lane / pieces, pc = lane - t * pieces;
            const int first = (s.x.lo / TK + s.tile + t_next + t) * TK + pc * piece_tokens;
            b.mine = t < b.tiles && first < s.x.seq && first + piece_tokens > s.x.lo;
            if (b.mine) phys = a.table[(size_t)s.r * a.width + (first >> bshift)];
            b.tok = first & (a.block - 1);
            b.row = s.h;
            t_next += b.tiles;
            if (t_next == s.tiles) { more = walk.next(s); t_next = 0; }
        };
        const auto resolve = [&]() {                               // its scales and its place in the pool
            if (!b.mine) return;
            if (phys < 0 || phys >= a.num_blocks) { dev_set_error(kv::ERR_BLOCK_ID); phys = 0; }
            const size_t unit = (size_t)phys * a.Hkv + b.row;
            b.ks = a.ks[unit];
            b.vs = a.vs[unit];
            b.row = (int)((unit * a.block + b.tok) / L::ROW_TOKENS);
        };
        look_up();
        resolve();
        while (b.tiles > 0 && ok) {
            const Batch now = b;
            look_up();
            for (int t = 0; t < now.tiles; t++) {
                if (used >= a.stages) {
                    if (!ptx::mbar_wait_warp(EMPTY(stage), phase ^ 1u)) { dev_set_error(ERR_WAIT | 1u); ok = false; break; }
                }
                const bool here = now.mine && lane / pieces == t;
                const int pc = lane - t * pieces;
                if (here) {
                    const float v1 = now.vs == 0.f ? 1.f : now.vs;
                    asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(scales_at + (stage * SLOT_SCALES + pc) * 16), "f"(now.ks), "f"(lg2(v1)),
                                 "f"(1.f / v1), "f"(now.vs == 0.f ? 1.f : 0.f) : "memory");
                }
                const unsigned count = __popc(__ballot_sync(0xffffffffu, here));
                __syncwarp();                                      // the scales are there before the arrival
                if (lane == 0) ptx::mbar_arrive_expect_tx(FULL(stage), count * 2u * (unsigned)(piece_tokens * D));
                if (here) {
                    const uint32_t at = ring_at + (uint32_t)stage * (uint32_t)S::STAGE_BYTES + (uint32_t)(pc * piece_tokens / L::ROW_TOKENS) * 128u;
#pragma unroll
                    for (int pl = 0; pl < L::PLANES; pl++) {
                        ptx::tma_load_2d(at + pl * L::PLANE_BYTES, &map_k, pl * 128, now.row, FULL(stage));
                        ptx::tma_load_2d(at + L::BYTES + pl * L::PLANE_BYTES, &map_v, pl * 128, now.row, FULL(stage));
                    }
                }
                used++;
                if (++stage == a.stages) { stage = 0; phase ^= 1u; }
            }
            resolve();
        }
        if (!ok) for (int i = 0; i < 64; i++) __nanosleep(50000);    // copies in flight end before the CTA's shared memory is another's
        return;
    }

    // ---- consumers ------------------------------------------------------------------------------------------------------------------
    const int g = lane >> 2, c = lane & 3;
    Walk walk(a, cum, u0, u1, ROWS);
    Segment s;
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    const float inf = __int_as_float(0x7f800000);
    while (walk.next(s)) {
        const int rows = min(ROWS, s.x.n * a.G - s.rg * ROWS);            // of this row group
        uint4 qf[QREG ? SETS * KS : 1];
        float fac[NR], B[NR], l[NR];
        int hi[NR], lo[NR];
        float acc[PM][NT][4];
        int min_hi = 0x7fffffff, max_lo = 0;
#pragma unroll
        for (int i = 0; i < NR; i++) {
            const int row = g + 8 * i, rho = s.rg * ROWS + row;
            const int query = min(rho / a.G, s.x.n - 1), at = s.x.seq - s.x.n + query;
            hi[i] = a.causal ? at : s.x.seq - 1;
            lo[i] = a.window > 0 ? at - a.window + 1 : 0;
            min_hi = min(min_hi, hi[i]);
            max_lo = max(max_lo, lo[i]);
            B[i] = -inf;
            l[i] = 0.f;
        }
        min_hi = __reduce_min_sync(0xffffffffu, min_hi);
        max_lo = __reduce_max_sync(0xffffffffu, max_lo);
        // Q: the row's largest magnitude, the digits.  Element order inside a step is the codes' order in memory: step k of lane column c is
        // elements 8 (k & 1) ... + 8 of its (k / 2)-th piece.
        const auto load_rows = [&](int i, uint4 *dst, int stride) {
            const int row = g + 8 * i, rho = s.rg * ROWS + row, query = rho / a.G, head = s.h * a.G + rho - query * a.G;
            const bool there = row < rows;
            const T *src = static_cast<const T *>(a.q) + (long long)(s.x.q0 + query) * a.ldq + (long long)head * D;
            float4 v[KS][2];
            float amax = 0.f;
#pragma unroll
            for (int k = 0; k < KS; k++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int d = L::qk_plane(k >> 1) * 128 + L::qk_piece(c, k >> 1) * 16 + (k & 1) * 8 + e * 4;
                    v[k][e] = there ? load4(src + d) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
#pragma unroll
            for (int k = 0; k < KS; k++)
#pragma unroll
                for (int e = 0; e < 2; e++)
                    amax = fmaxf(fmaxf(amax, fmaxf(fabsf(v[k][e].x), fabsf(v[k][e].y))), fmaxf(fabsf(v[k][e].z), fabsf(v[k][e].w)));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            // the row in units of its last digit: amax becomes 127 * 128^2; by a power of two first, so that neither factor leaves fp32
            constexpr float top = 127.f * 16384.f;
            const float p2 = row_factor(amax), f = amax > 0.f ? top / (amax * p2) : 1.f;
            float bad = 0.f;                                           // NaN if an element is not a number or infinite: the digits cannot tell
#pragma unroll
            for (int k = 0; k < KS; k++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float4 &x = v[k][e];
                    bad += (x.x * 0.f + x.y * 0.f) + (x.z * 0.f + x.w * 0.f);
                    x.x = x.x * p2 * f; x.y = x.y * p2 * f; x.z = x.z * p2 * f; x.w = x.w * p2 * f;
                }
            bad += __shfl_xor_sync(0xffffffffu, bad, 1);
            bad += __shfl_xor_sync(0xffffffffu, bad, 2);
            const float back = a.scale * (a.softcap > 0.f ? 1.f / a.softcap : LOG2E) / f / p2 + bad;
            if constexpr (QREG) fac[i] = back;
            else if (c == 0) row_fac[row] = back;
#pragma unroll
            for (int k = 0; k < KS; k++) {
                const uint32_t a0 = digit4(v[k][0], 16384.f, 1.f / 16384.f), a2 = digit4(v[k][1], 16384.f, 1.f / 16384.f);
                const uint32_t a1 = digit4(v[k][0], 128.f, 1.f / 128.f), a3 = digit4(v[k][1], 128.f, 1.f / 128.f);
                dst[(i * KS + k) * stride] = make_uint4(a0, a1, a2, a3);
                const uint32_t b0 = digit4(v[k][0], 1.f, 1.f), b1 = digit4(v[k][1], 1.f, 1.f);
                uint32_t *third = reinterpret_cast<uint32_t *>(dst + ((NR + (i >> 1)) * KS + k) * stride);
                third[i & 1] = b0;                                     // row g: first of the pairs, row g + 8: second
                third[2 + (i & 1)] = b1;
                if (NR == 1) { third[1] = 0u; third[3] = 0u; }
            }
        };
        if constexpr (QREG) {
#pragma unroll
            for (int i = 0; i < NR; i++) load_rows(i, qf, 1);
        } else {
            if (warp < NR) load_rows(warp, qs + lane, 32);
            asm volatile("bar.sync 1, %0;" ::"r"(CW * 32) : "memory");
#pragma unroll
            for (int i = 0; i < NR; i++) fac[i] = row_fac[g + 8 * i];
        }

#pragma unroll
        for (int mt = 0; mt < PM; mt++)
#pragma unroll
            for (int j = 0; j < NT; j++) acc[mt][j][0] = acc[mt][j][1] = acc[mt][j][2] = acc[mt][j][3] = 0.f;
        for (int t = 0; t < s.tiles; t++) {
            if (ok && !ptx::mbar_wait_warp(FULL(stage), phase)) { if (lane == 0) dev_set_error(ERR_WAIT | 2u); ok = false; }
            const int key0 = (s.x.lo / TK + s.tile + t) * TK + warp * 16;
            if (ok && key0 < s.x.seq && key0 + 16 > s.x.lo) {
                const uint32_t kt = ring_at + (uint32_t)stage * (uint32_t)S::STAGE_BYTES, vt = kt + L::BYTES;
                const float4 sc = lds_f4(scales_at + (stage * SLOT_SCALES + ((warp * 16) >> pshift)) * 16);
                int dot[SETS][2][4];
#pragma unroll
                for (int mt = 0; mt < SETS; mt++)
#pragma unroll
                    for (int i = 0; i < 2; i++) dot[mt][i][0] = dot[mt][i][1] = dot[mt][i][2] = dot[mt][i][3] = 0;
#pragma unroll
                for (int pq = 0; pq < L::STEPS; pq++) {
                    uint4 w[2];
#pragma unroll
                    for (int i = 0; i < 2; i++) w[i] = lds128(kt + L::piece(warp * 16 + L::token(i, g), L::qk_piece(c, pq), L::qk_plane(pq)));
#pragma unroll
                    for (int mt = 0; mt < SETS; mt++)
#pragma unroll
                        for (int k = 0; k < 2; k++) {
                            uint4 qa;
                            if constexpr (QREG) qa = qf[mt * KS + pq * 2 + k];
                            else qa = qs[(mt * KS + pq * 2 + k) * 32 + lane];
#pragma unroll
                            for (int i = 0; i < 2; i++) mma_s8(dot[mt][i], qa, k ? w[i].z : w[i].x, k ? w[i].w : w[i].y);
                        }
                }
                // scores in base 2, weights
                const bool edge = key0 + 15 > min_hi || key0 < max_lo || key0 + 15 >= s.x.seq;
                float x[NR][4];
                bool again = false;
                const auto scores = [&](int i, float (&y)[4]) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float d = fmaf((float)dot[i][e >> 1][e & 1], 16384.f,
                                             (float)(dot[i][e >> 1][2 + (e & 1)] * 128 + dot[NR + (i >> 1)][e >> 1][2 * (i & 1) + (e & 1)]));
                        y[e] = d;
                    }
                    const float f = fac[i] * sc.x;
                    if (a.softcap > 0.f) {
#pragma unroll
                        for (int e = 0; e < 4; e++) y[e] = capped(y[e] * f, a.softcap) + sc.y;
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; e++) y[e] = fmaf(y[e], f, sc.y);
                    }
                    if (edge) {
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const int key = key0 + L::token(e >> 1, 2 * c + (e & 1));
                            if (key > hi[i] || key < lo[i] || key >= s.x.seq) y[e] = -inf;
                        }
                    }
                };
                float top[NR];
#pragma unroll
                for (int i = 0; i < NR; i++) {
                    scores(i, x[i]);
                    top[i] = fmaxf(fmaxf(x[i][0], x[i][1]), fmaxf(x[i][2], x[i][3]));
                    again = again || top[i] > B[i] + 15.f;
                }
                if (__any_sync(0xffffffffu, again)) {
                    // a weight would pass 2^15: the rows' references move to where their largest is 2^8
#pragma unroll
                    for (int i = 0; i < NR; i++) {
                        float m = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
                        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                        const float now = m > B[i] + 8.f ? m - 8.f : B[i];
                        const float shrink = B[i] == -inf ? 1.f : ex2(B[i] - now);        // nothing is summed while B is -inf
                        B[i] = now;
                        l[i] *= shrink;
#pragma unroll
                        for (int j = 0; j < NT; j++) {
                            if constexpr (SPLIT) { acc[i][j][0] *= shrink; acc[i][j][1] *= shrink; acc[i][j][2] *= shrink; acc[i][j][3] *= shrink; }
                            else { acc[i >> 1][j][2 * (i & 1)] *= shrink; acc[i >> 1][j][2 * (i & 1) + 1] *= shrink; }
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < NR; i++) {
                    const float ref = B[i] == -inf ? 0.f : B[i];
#pragma unroll
                    for (int e = 0; e < 4; e++) x[i][e] = edge && x[i][e] == -inf ? 0.f : ex2(x[i][e] - ref);
                    l[i] = fmaf((x[i][0] + x[i][1]) + (x[i][2] + x[i][3]), sc.z, l[i]);
                }
                if (sc.w != 0.f) {
#pragma unroll
                    for (int i = 0; i < NR; i++) x[i][0] = x[i][1] = x[i][2] = x[i][3] = 0.f;
                }
                uint4 pa[PM];
#pragma unroll
                for (int mt = 0; mt < PM; mt++) {
                    const int i = SPLIT ? mt : 2 * mt;
                    const __half2 h0 = __floats2half2_rn(x[i][0], x[i][1]), h1 = __floats2half2_rn(x[i][2], x[i][3]);
                    if constexpr (SPLIT) {
                        const float2 f0 = __half22float2(h0), f1 = __half22float2(h1);
                        pa[mt] = make_uint4(h2_bits(h0), h2_bits(__floats2half2_rn(x[i][0] - f0.x, x[i][1] - f0.y)),
                                            h2_bits(h1), h2_bits(__floats2half2_rn(x[i][2] - f1.x, x[i][3] - f1.y)));
                    } else {
                        constexpr int o = NR > 1 ? 1 : 0;
                        pa[mt] = make_uint4(h2_bits(h0), o ? h2_bits(__floats2half2_rn(x[i + o][0], x[i + o][1])) : 0u,
                                            h2_bits(h1), o ? h2_bits(__floats2half2_rn(x[i + o][2], x[i + o][3])) : 0u);
                    }
                }
                // values: lane row g holds the 16 (dim 64: 8) elements of a piece, one for each group of eight columns
#pragma unroll
                for (int pl = 0; pl < L::PLANES; pl++) {
                    uint32_t v[4][4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const int tok = warp * 16 + L::token(k >> 1, 2 * c + (k & 1));
                        if constexpr (D == 64) {
                            const uint2 w = lds64(vt + L::piece(tok, g >> 1, 0) + (g & 1) * 8);
                            v[k][0] = w.x; v[k][1] = w.y;
                        } else {
                            const uint4 w = lds128(vt + L::piece(tok, g, pl));
                            v[k][0] = w.x; v[k][1] = w.y; v[k][2] = w.z; v[k][3] = w.w;
                        }
                    }
#pragma unroll
                    for (int w = 0; w < (D == 64 ? 2 : 4); w++) {
                        const uint32_t a0 = v[0][w] ^ 0x80808080u, a1 = v[1][w] ^ 0x80808080u, a2 = v[2][w] ^ 0x80808080u, a3 = v[3][w] ^ 0x80808080u;
                        const uint32_t e0 = __byte_perm(a0, a1, 0x5140), o0 = __byte_perm(a0, a1, 0x7362);
                        const uint32_t e1 = __byte_perm(a2, a3, 0x5140), o1 = __byte_perm(a2, a3, 0x7362);
                        const uint32_t b[4][2] = {{codes_f16<0x4140>(e0), codes_f16<0x4140>(e1)}, {codes_f16<0x4342>(e0), codes_f16<0x4342>(e1)},
                                                  {codes_f16<0x4140>(o0), codes_f16<0x4140>(o1)}, {codes_f16<0x4342>(o0), codes_f16<0x4342>(o1)}};
#pragma unroll
                        for (int j = 0; j < 4; j++)
#pragma unroll
                            for (int mt = 0; mt < PM; mt++) mma_f16(acc[mt][pl * 16 + w * 4 + j], pa[mt], b[j][0], b[j][1]);
                    }
                }
            }
            __syncwarp();
            if (ok && lane == 0) ptx::mbar_arrive(EMPTY(stage));
            if (++stage == a.stages) { stage = 0; phase ^= 1u; }
        }

        // ---- the warps meet --------------------------------------------------------------------------------------------------------
#pragma unroll
        for (int i = 0; i < NR; i++) {
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
            if (c == 0) ml[warp * ROWS + g + 8 * i] = make_float2(B[i], l[i]);
        }
        asm volatile("bar.sync 1, %0;" ::"r"(CW * 32) : "memory");
#pragma unroll
        for (int i = 0; i < NR; i++) {
            const int row = g + 8 * i;
            float top = ml[row].x;
#pragma unroll
            for (int w = 1; w < CW; w++) top = fmaxf(top, ml[w * ROWS + row].x);
            const float f = B[i] == -inf ? 0.f : ex2(B[i] - top);
            float4 *dst = reinterpret_cast<float4 *>(meet + ((size_t)warp * ROWS + row) * D);
            if (row < rows) {
#pragma unroll
                for (int pl = 0; pl < L::PLANES; pl++)
#pragma unroll
                    for (int half = 0; half < 2; half++)
#pragma unroll
                        for (int k = 0; k < (D == 64 ? 2 : 4); k++) {
                            float o[4];
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                const float *q4 = acc[SPLIT ? i : i >> 1][pl * 16 + 4 * k + e];
                                o[e] = (SPLIT ? q4[half] + q4[2 + half] : q4[2 * (i & 1) + half]) * f;
                            }
                            const int f4 = D == 64 ? 4 * c + 2 * half + k : 32 * pl + 8 * c + 4 * half + k;
                            dst[meet_pos<D>(f4, row)] = make_float4(o[0], o[1], o[2], o[3]);
                        }
            }
        }
        asm volatile("bar.sync 1, %0;" ::"r"(CW * 32) : "memory");
        const bool whole = s.tiles == s.pair_tiles;
        const int slot = 2 * (int)cta + (s.tile == 0 ? 1 : 0);
        const auto finish = [&](int row, int f4, float4 v, float top, float sum) {     // v: the weighted values, sum: the weights'
            const int rho = s.rg * ROWS + row, query = rho / a.G, head = s.h * a.G + rho - query * a.G;
            const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);        // nothing seen: zeros
            v.x *= inv; v.y *= inv; v.z *= inv; v.w *= inv;
            store4(static_cast<T *>(a.out) + (long long)(s.x.q0 + query) * a.ldo + (long long)head * D + 4 * f4, v);
            if (a.lse && f4 == 0) a.lse[(size_t)(s.x.q0 + query) * a.Hq + head] = sum > 0.f ? (top + log2f(sum)) * LN2 : (sum == 0.f ? -inf : sum);
        };
        for (int e = tid; e < rows * (D / 4); e += CW * 32) {
            const int row = e / (D / 4), f4 = e - row * (D / 4);
            float top = ml[row].x, sum = 0.f;
#pragma unroll
            for (int w = 1; w < CW; w++) top = fmaxf(top, ml[w * ROWS + row].x);
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < CW; w++) {
                const float2 x = ml[w * ROWS + row];
                const float4 o = reinterpret_cast<const float4 *>(meet + ((size_t)w * ROWS + row) * D)[meet_pos<D>(f4, row)];
                sum += x.x == -inf ? 0.f : x.y * ex2(x.x - top);
                v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
            }
            if (whole) finish(row, f4, v, top, sum);
            else {
                reinterpret_cast<float4 *>(a.part + ((size_t)slot * ROWS + row) * D)[f4] = v;
                if (f4 == 0) a.part_ml[(size_t)slot * ROWS + row] = make_float2(top, sum);
            }
        }
        if (whole) continue;
        // ---- the CTAs that share the pair meet: the last to come joins, in the order of the ranges ----------------------------------------
        const unsigned c0 = cta_of((unsigned)s.pair0), c1 = cta_of((unsigned)(s.pair0 + s.pair_tiles - 1));
        __threadfence();
        asm volatile("bar.sync 1, %0;" ::"r"(CW * 32) : "memory");
        if (tid == 0) {
            const unsigned seen = atomicAdd(a.count + c0, 1u);
            last_flag = seen == c1 - c0;
            if (seen == c1 - c0) a.count[c0] = 0u;                 // as the next call expects it
        }
        asm volatile("bar.sync 1, %0;" ::"r"(CW * 32) : "memory");
        if (last_flag) {
            __threadfence();
            for (int e = tid; e < rows * (D / 4); e += CW * 32) {
                const int row = e / (D / 4), f4 = e - row * (D / 4);
                float top = -inf, sum = 0.f;
                const auto at = [&](unsigned k) { return (size_t)(2 * k + (k == c0 ? 1 : 0)) * ROWS + row; };
#pragma unroll 4
                for (unsigned k = c0; k <= c1; k++) top = fmaxf(top, __ldcg(&a.part_ml[at(k)]).x);
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
                for (unsigned k = c0; k <= c1; k++) {
                    const float2 x = __ldcg(&a.part_ml[at(k)]);
                    const float4 o = __ldcg(reinterpret_cast<const float4 *>(a.part + at(k) * D) + f4);
                    const float f = x.x == -inf ? 0.f : ex2(x.x - top);
                    sum += x.y * f;
                    v.x += o.x * f; v.y += o.y * f; v.z += o.z * f; v.w += o.w * f;
                }
                finish(row, f4, v, top, sum);
            }
        }
        asm volatile("bar.sync 1, %0;" ::"r"(CW * 32) : "memory");          // last_flag has been read
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------------
struct Call {
    Args a;
    const int8_t *k, *v;
    int dtype, dim;
};

// Workspace: the arrival counts, then the partial results of 2 ranges' ends per CTA.  32 rows at most.
constexpr int MAX_CTAS_PER_SM = 3, MAX_ROWS = 32;
inline size_t count_bytes() { return ((size_t)sm_count() * MAX_CTAS_PER_SM * 4 + 255) & ~(size_t)255; }
inline size_t workspace_bytes(int dim) {
    const size_t slots = (size_t)sm_count() * MAX_CTAS_PER_SM * 2;
    return count_bytes() + slots * MAX_ROWS * 8 + slots * MAX_ROWS * dim * 4;
}

template <typename T, int D, int R>
inline int launch_t(Call &c, cudaStream_t st) {
    using S = Shape<T, D, R>;
    Args &a = c.a;
    constexpr int per_sm = S::PER_SM;
    a.stages = S::stages(a.R);
    const size_t smem = S::fixed_bytes(a.R) + a.stages * S::STAGE_BYTES;
    auto kern = attention_q8_kernel<T, D, R>;
    static PerDevice<size_t> configured_dev;
    size_t &configured = configured_dev.get();
    if (smem > configured) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return cuda_fail(e, "attention_q8 smem opt-in");
        configured = smem;
    }
    const uint64_t row = D == 256 ? 256 : 128, rows = (uint64_t)a.num_blocks * a.Hkv * a.block * D / row;
    const uint32_t box = (uint32_t)((a.block < TK ? a.block : TK) / Tile<D>::ROW_TOKENS);
    CUtensorMap mk, mv;
    int rc = tmap_cached(&mk, c.k, row, rows, 128, box, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B);
    if (rc == W4A8_OK) rc = tmap_cached(&mv, c.v, row, rows, 128, box, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B);
    if (rc != W4A8_OK) return rc;
    const int sms = sm_count();
    cudaError_t e = launch_pdl(kern, dim3(sms * per_sm), dim3(THREADS), smem, st, mk, mv, a);
    return e == cudaSuccess ? launch_status("attention_q8") : cuda_fail(e, "attention_q8 launch");
}

template <typename T, int D>
inline int launch_r(Call &c, int rows, cudaStream_t st) {
    constexpr int most = (std::is_same<T, float>::value ? 8 : 16) * (D == 256 ? 1 : 2);     // the registers' limit
    if (rows <= 8) return launch_t<T, D, 8>(c, st);
    if (rows <= 16 || most == 16) return launch_t<T, D, most < 16 ? most : 16>(c, st);
    return launch_t<T, D, most>(c, st);
}
template <typename T>
inline int launch_d(Call &c, int rows, cudaStream_t st) {
    if (c.dim == 64) return launch_r<T, 64>(c, rows, st);
    if (c.dim == 128) return launch_r<T, 128>(c, rows, st);
    return launch_r<T, 256>(c, rows, st);
}

// `rows`: queries x heads of a group of the request with most of them.
inline int launch(Call &c, int rows, cudaStream_t st) {
    const Args all = c.a;
    for (int r0 = 0; r0 < all.R; r0 += MAX_R) {                    // requests beyond MAX_R: further launches
        c.a = all;
        c.a.R = all.R - r0 < MAX_R ? all.R - r0 : MAX_R;
        c.a.cu_q = all.cu_q + r0;
        c.a.seq_len = all.seq_len + r0;
        c.a.table = all.table + (size_t)r0 * all.width;
        int rc = c.dtype == W4A8_F32 ? launch_d<float>(c, rows, st) : c.dtype == W4A8_F16 ? launch_d<__half>(c, rows, st) : launch_d<__nv_bfloat16>(c, rows, st);
        if (rc != W4A8_OK) return rc;
    }
    return W4A8_OK;
}

}  // namespace attn
}  // namespace w4a8
