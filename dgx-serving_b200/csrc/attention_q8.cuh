// Attention of few queries a request over the 8-bit paged KV cache: a stream of the blocks through the tensor cores, which take the codes as they are.
//
//   s[i,j] = scale * ks[block(j)] * sum_d q[i,d] K[j,d]           (K, V: the int8 codes)
//   o[i]   = sum_j exp(s[i,j] - m) vs[block(j)] V[j] / sum_j exp(s[i,j] - m),   j over what query i sees
//
// What bounds it: the codes have to come from HBM once, 2 * dim bytes a token and kv head.  Everything else is arranged not to be in the way:
//  - Work is cut evenly: the (request, kv head, row group) pairs' key tiles of 128 tokens, laid one behind the other, are divided into equal
//    ranges, one per SM, whatever the lengths.  A pair that several CTAs share leaves partial results (reference, sum, weighted values) in the
//    workspace; neighbours are joined by the last of them to finish, in the order of the ranges, so the result does not depend on who is last.
//    One launch.
//  - Both products are tcgen05.mma kind::i8 with the keys' tile as the 128-row operand, so the codes go from HBM by TMA to shared memory (128-byte
//    swizzle; along the block table, a block never has to be a whole tile) and no thread touches them: S^T [keys][rows] = K Q^T with K as it
//    lies, O^T [dim][rows] += V^T P^T with V read as the transposed operand.  Widening the codes to fp16 for mma.sync cost 450 instructions for 16
//    keys and bound the stream: two requests of 115k tokens 96 us, 64 ragged ones of up to 8192 tokens 128.  Now 84 us (5.9 TB/s) and 101 (5.4).
//  - A query row is a fixed-point number relative to its largest magnitude, three signed digits of base 256 (2^-23 of it): three columns.  A weight
//    times its block's scale is a whole number too, x = exp(s) 2^-A * vs 2^-E * 2^25 up to 2^31, four columns of P.  All sums are whole numbers and
//    exact; O stays in tensor memory over the tiles.  The row's reference A is such that its largest weight was in [1, 2) when it was chosen, E is the
//    largest exponent of the scales of blocks that the row has seen of.  When a weight would pass 2^4.9 or E grows, O is read out, rescaled and summed in
//    fp32.  So a weight times its scale is rounded to 2^-26 of the row's largest of either, or as fp32 is; A and E are whole numbers and rescaling is
//    exact.  The sum of the weights, l = sum exp(s) 2^-A, knows nothing of the scales.  (One reference for the products, 2^28 for the largest, with l
//    taken from them by 1 / vs, took 51.5, 40.4 and 98.9 us where few queries, a window and ragged tokens now take 53.5, 43 (two of it the caps) and 100.8; but l left fp32
//    at scales above 2^62, and lost the weights of tokens whose scale is 2^-150 of another's.)
//  - 128 threads have a key each, about thirty instructions for a row.  Two such groups take the tiles in turn, each with its own S, P, O, reference and
//    sums, because a tile's chain of steps (1300 cycles with 4 rows, 3500 with 16) takes longer than its bytes do; they meet at the end of a pair, one
//    handing over, the other writing.
//  - What is left: 3 us before the first tile and 3 us for the last join, and for many rows the chain: 16 requests of up to 56 rows and 6000 tokens take
//    54 us where their bytes take 9.
#pragma once
#include "kv_cache.cuh"
#include "ptx_sm100.cuh"
#include "tmap_cache.cuh"

namespace w4a8 {
namespace attn {

constexpr int TK = 128;                    // keys of a tile
constexpr int THREADS = 384;               // warps 0-3, 4-7: a key (then a dim) a thread; 8, 9: copies of K, of V; 10: products; 11: queries
constexpr int MAX_R = 2048;                // requests of one launch (their sums lie in shared memory)
constexpr int FEW_ROWS = 64;               // rows (queries x heads of a group) of a request that this kernel takes at most: half a row tile of the other
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr unsigned ERR_WAIT = 0xA00u;
// log2 of a weight's whole number when A is chosen, and of a weight before A moves: with a scale's mantissa in [1, 2) they make 30.9, and four signed
// digits reach 2^30.99.  (27 and 2.9 move A more often: 1.7 us more of 54.)
constexpr float TOP = 25.f, LIMIT = 4.9f;
constexpr float NONE = -1e30f;             // A before a key was seen
constexpr int START = 4;                   // tiles whose time beginning and ending a pair takes (64 ragged requests: 104.5 us with 1, 99.3 with 4, 100.7 with 6)
constexpr int FLUSH = 900;                 // tiles after which O is read out at the latest: 128 * 128 * 127 * 900 < 2^31

struct Args {
    const void *q;
    void *out;
    float *lse;
    const float *ks, *vs;
    const int32_t *table, *cu_q, *seq_len;
    long long ldq, ldo;
    int R, T, width, Hq, Hkv, G, block, num_blocks, k_stages, v_stages;
    int causal, window;
    float scale, softcap;
    int few;                               // rows (queries * G) of a request that this kernel takes at most; more are another kernel's
    // workspace, by a CTA's two ends: arrivals, zero between calls; [2 * CTAs][rows] A, E, sum; [2 * CTAs][rows][dim] values; groups of CTAs alike
    unsigned *count, *count2;
    float4 *part_ml, *part2_ml;
    float *part, *part2;
};

__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }          // -126 <= e <= 127
// The exponent of a scale (0 and what is not a number: that of the smallest there are).
constexpr int LEAST = -150;
__device__ __forceinline__ int exponent_of(float vs) {
    const int e = (int)(__float_as_uint(vs) >> 23) - 127;
    return !(vs > 0.f && vs < __int_as_float(0x7f800000)) ? LEAST : e > -127 ? e : (int)(__float_as_uint(vs * 0x1p64f) >> 23) - 127 - 64;
}
// 2^d for a whole number d, -250 <= d <= 250, as a product of two powers of two.
__device__ __forceinline__ float2 pow2_parts(int d) { return make_float2(pow2(d >> 1), pow2(d - (d >> 1))); }

// ---- which keys and how much work ----------------------------------------------------------------------------------------------------
struct Request {
    int q0, n, seq, lo, tiles, groups;       // first row of Q, rows, tokens, first token that any row sees, tiles from its tile on, row groups
};
// The first key that the query at position `pos` sees.  (One in front of all tokens sees as much as the first; so no difference leaves 32 bits.)
__device__ __forceinline__ int first_seen(int pos, int window) { return window > 0 ? max(0, max(pos, 0) - window + 1) : 0; }
__device__ __forceinline__ Request request(const Args &a, int r, int rows_per_group) {
    Request x;
    x.q0 = max(0, min(a.cu_q[r], a.T));
    x.n = max(0, min(a.cu_q[r + 1], a.T) - x.q0);
    x.seq = max(0, a.seq_len[r]);
    const long long most = min((long long)a.width * a.block, (long long)kv::LONGEST);
    if (x.seq > most) { x.seq = (int)most; dev_set_error(kv::ERR_LENGTH); }
    x.lo = first_seen(x.seq - x.n, a.window);
    // at least one tile, so that rows that see nothing are written too
    x.tiles = x.seq > x.lo ? (x.seq + TK - 1) / TK - x.lo / TK : 1;
    const int rows = x.n * a.G;
    x.groups = rows <= a.few ? (rows + rows_per_group - 1) / rows_per_group : 0;
    return x;
}

// Units: a pair is START of them and one for each of its tiles, because beginning and ending a pair costs a CTA as much as START tiles; a bound
// that falls into the START lies in front of the first tile.  A CTA's range cut at the pairs' ends:
struct Segment {
    int r, h, rg, tile, tiles;               // tiles [tile, tile + tiles) of the pair's
    int pair0, pair_tiles;                   // the unit of the pair's first tile, its tiles
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
        const unsigned span = (unsigned)(x.tiles + START), in = u - cum[r], pair = in / span, tile0 = cum[r] + pair * span + START;
        const unsigned t = u > tile0 ? u - tile0 : 0, t1 = end > tile0 ? min(end - tile0, (unsigned)x.tiles) : 0;
        u = tile0 + x.tiles;
        if (t1 <= t) return false;
        s.r = r;
        s.h = (int)(pair % (unsigned)a.Hkv);
        s.rg = (int)(pair / (unsigned)a.Hkv);
        s.tile = (int)t;
        s.tiles = (int)(t1 - t);
        s.pair0 = (int)tile0;
        s.pair_tiles = x.tiles;
        s.x = x;
        return true;
    }
};

__device__ __forceinline__ void sts128(uint32_t addr, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
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
// Power of two that brings a row whose largest magnitude is amax near 2^13; 1 for zeros and what is no number.
__device__ __forceinline__ float row_factor(float amax) {
    if (!(amax > 0.f) || !(amax < __int_as_float(0x7f800000))) return 1.f;
    int e = 13 - (((__float_as_int(amax) >> 23) & 0xFF) - 127);
    e = max(-126, min(126, e));
    return __int_as_float((e + 127) << 23);
}

__device__ __forceinline__ float warp_max(float x) { float y; asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float lg2(float x) { float y; asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
// cap * tanh(x) * log2 e with x in units of cap.  tanh x = 1 - 2 / (1 + e^2x) has the error of a number near 1, so for |x| up to 0.625 it is x + x^3 p(x^2)
// instead, p of degree 3 and with the least largest relative error (2^-22.97; fitted by reweighted least squares).  Either way the score is off by 2^-21
// of itself.  (One quotient of polynomials for all x, degrees 4 and 4, took 468 us for a prompt of 4096 where both of these, each element choosing, take
// 386 and the first, two elements at a time where a warp has no others, 301; the second alone 371.)  And `add`.
constexpr float SMALL_X = 0.625f, TANH3 = -0.3333234190940857f, TANH5 = 0.13308174908161163f, TANH7 = -0.051947902888059616f, TANH9 = 0.015195372514426708f;
__device__ __forceinline__ float capped(float x, float cap, float add) {
    const float u = x * x, p = fmaf(fmaf(fmaf(TANH9, u, TANH7), u, TANH5), u, TANH3);
    const float t = fabsf(x) <= SMALL_X ? fmaf(x * u, p, x) : 1.f - __fdividef(2.f, 1.f + ex2(x * (2.f * LOG2E)));
    return fmaf(cap * LOG2E, t, add);
}

// Bounded waits without a call: a kernel that moves registers between its warps cannot have one.
__device__ __forceinline__ bool wait_one(uint32_t bar, uint32_t parity) {
    if (ptx::mbar_try_wait(bar, parity)) return true;
    long long since = 0;
#pragma unroll 1
    for (;;) {
#pragma unroll 1
        for (int i = 0; i < 64; i++)
            if (ptx::mbar_try_wait(bar, parity)) return true;
        const long long now = clock64();
        if (since == 0) since = now;
        else if (now - since > (1ll << 28)) return false;
    }
}
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity) {
    const bool ok = wait_one(bar, parity);
    return __all_sync(0xffffffffu, ok);
}
__device__ __forceinline__ bool test_one(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    return done != 0;
}
// The same for a warp that waits long: it sleeps between the attempts and leaves the issue slots to the others.
__device__ __forceinline__ bool wait_idle(uint32_t bar, uint32_t parity) {
    bool ok = ptx::mbar_try_wait(bar, parity);
#pragma unroll 1
    for (int i = 0; i < (1 << 21) && !ok; i++) {
        __nanosleep(100);
        ok = ptx::mbar_try_wait(bar, parity);
    }
    return __all_sync(0xffffffffu, ok);
}
// What the warps have to know of a segment, left by the one that prepares its queries.  tiles 0: there is no further one.
struct Work { int tiles, tile0, min_hi, max_lo, n, q0, rg, h, first, pair0, pair_tiles, pad; };   // keys up to min_hi and from max_lo on: every row sees them
constexpr int WORKS = 4;
constexpr int FAN = 16, MAX_ROWS = 16;     // CTAs whose partial results are joined at a time; rows of a partial result

// ---- operands ------------------------------------------------------------------------------------------------------------------------------
// A tile of codes: planes of 128-byte rows, the 16-byte piece c of row r at c ^ (r & 7).  dim 128 and 256: a row is a token, a plane 128 elements.
// dim 64: K in rows of 64 bytes (piece c of row r at c ^ (r >> 1 & 3)); V in rows of two tokens, so that the instruction's 128 rows are (token's
// parity, element), the keys of the product pairs of tokens, and the weights' columns come twice, for the even and the odd tokens: half of what
// the instruction sums is the wrong parity's and is not read.
template <int D> struct Tile {
    static constexpr int PLANES = D == 256 ? 2 : 1, BYTES = TK * D, PLANE_BYTES = BYTES / PLANES;
    static constexpr int K_ROW = D == 64 ? 64 : 128, V_TOKENS = D == 64 ? 2 : 1;             // bytes of a row of K, tokens of a row of V
};
// K-major operand of `ROW`-byte rows: 8 rows ROW * 8 bytes; swizzle mode 2 (128 bytes) or 4 (64 bytes).
template <int ROW> __device__ __forceinline__ uint64_t desc_k(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (1ull << 16) | ((uint64_t)(ROW * 8 >> 4) << 32) | (1ull << 46) | ((ROW == 128 ? 2ull : 4ull) << 61);
}
// MN-major operand of 128 bytes: a row of 128 elements for each k, 8 of them 1024 bytes.
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (1ull << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// The same of W bytes, all of the operand's N (W 16: not swizzled; else W bytes).
template <int W> __device__ __forceinline__ uint64_t desc_p(uint32_t addr) {
    constexpr uint64_t stride = W * 8 >> 4, mode = W == 128 ? 2 : W == 64 ? 4 : W == 32 ? 6 : 0;
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (stride << 16) | (stride << 32) | (1ull << 46) | (mode << 61);
}
// D = int32, A and B signed bytes, 128 rows, N columns; bits 15 and 16: A and B are MN-major.
__host__ __device__ constexpr uint32_t idesc_s8(int N, int mn) { return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(mn * 3) << 15) | ((uint32_t)(N >> 3) << 17) | (8u << 24); }
using ptx::elected;
using ptx::umma_commit;
using ptx::umma_s8;
__device__ __forceinline__ float out_round(float, float v) { return v; }
__device__ __forceinline__ __half out_round(__half, float v) { return __float2half_rn(v); }
__device__ __forceinline__ __nv_bfloat16 out_round(__nv_bfloat16, float v) { return __float2bfloat16_rn(v); }
// N columns of tensor memory of this lane, on their way until columns_arrived.
template <int N> __device__ __forceinline__ void columns_load(uint32_t addr, uint32_t (&v)[N]) {
    if constexpr (N == 12) {
        ptx::tmem_ld(addr, *reinterpret_cast<uint32_t(*)[8]>(v));
        ptx::tmem_ld(addr + 8, *reinterpret_cast<uint32_t(*)[4]>(v + 8));
    } else if constexpr (N == 24) {
        ptx::tmem_ld(addr, *reinterpret_cast<uint32_t(*)[16]>(v));
        ptx::tmem_ld(addr + 16, *reinterpret_cast<uint32_t(*)[8]>(v + 16));
    } else ptx::tmem_ld(addr, v);
}
template <int N> __device__ __forceinline__ void columns_arrived(uint32_t (&v)[N]) {
    ptx::tmem_ld_wait();
#pragma unroll
    for (int c = 0; c < N; c++) asm volatile("" : "+r"(v[c]));        // nothing that reads them moves in front of the wait
}

// R rows (queries x heads of a group): 3 columns of S and 4 of P for each, in whole sixteens.
template <int D, int R_> struct Shape {
    static constexpr int R = R_, N = (3 * R + 15) / 16 * 16, NP = 4 * R, DP = D == 256 ? 2 : 1, OC = D == 64 ? 2 * NP : DP * NP;    // DP: dims of a thread; OC: columns of O
    static constexpr int P_ROW = D == 64 ? 2 * NP : NP;                              // bytes of P of a token (dim 64: of a pair of tokens)
    static constexpr int STAGE = Tile<D>::BYTES, QB = N * D, PB = NP * TK;             // a stage: a tile of K or of V
    static constexpr int SCALES = 8;                                                   // blocks of a tile at most
    // K may leave as soon as its product is issued, V only when its weights are.  At dim 256 there are five stages in all, and K's leave early (requests with a
    // window of 1024 tokens 44.7 -> 40.1 us); at the others K's loads would then run ahead of V's (two of 115k tokens 83.7 -> 87), so both leave together.
    static constexpr bool EARLY = D == 256;
    static constexpr int MAX_STAGES = 8, SLOTS = 16;                                   // of each side; tiles' scales, more than are between copy and scores
    static constexpr int FIXED = 1024 + 2 * QB + 2 * PB + 1024 + SLOTS * SCALES * 16 + 2 * R * 16 + 2 * 4 * R * 4 + R * 16 + 2 * R * 24 + R * (D == 64 ? 128 : D) * 4 + 2 * (FAN + 3) * MAX_ROWS * 4;   // and 4 bytes a request
    static inline int fixed_bytes(int n) { return (FIXED + (n + 4) * 4 + 1023) & ~1023; }
    static inline int stages(int n) {                                                  // of both sides together
        const int k = (226 * 1024 - fixed_bytes(n)) / STAGE;
        return k < 2 * MAX_STAGES ? k : 2 * MAX_STAGES;
    }
    static_assert(NP % 16 == 0 && 2 * N + 2 * OC <= 512 && FIXED + (MAX_R + 4) * 4 + 1024 + 4 * STAGE <= 226 * 1024, "shape");
};

// CAP: scores are capped.  (In one kernel their code cost the others 3 us of 54 with many rows.)
template <typename T, int D, int R, bool CAP>
__global__ void __launch_bounds__(THREADS, 1) attention_q8_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Args a) {
    using S = Shape<D, R>;
    using L = Tile<D>;
    constexpr int N = S::N, NP = S::NP, DP = S::DP;
    extern __shared__ unsigned char smem_raw[];
    // ring, Q and P first (1024-byte aligned for the swizzle), then the rest
    unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char *p = smem + (size_t)(a.k_stages + a.v_stages) * S::STAGE;
    unsigned char *qs = p; p += 2 * S::QB;
    unsigned char *ps = p; p += 2 * S::PB;
    unsigned char *control = p; p += 1024;
    float4 *scales = reinterpret_cast<float4 *>(p); p += S::SLOTS * S::SCALES * 16;   // a tile's blocks: ks; vs; their largest exponent (below); 0, or not a number where vs is none
    float4 *rec = reinterpret_cast<float4 *>(p); p += 2 * R * 16;                          // a row's factor, -, last and first key (as int)
    float4 *over_ml = reinterpret_cast<float4 *>(p); p += R * 16;                          // what one group hands over: A, E, sum; values
    float *reds = reinterpret_cast<float *>(p); p += 2 * 4 * R * 4;
    float *refs = reinterpret_cast<float *>(p); p += 2 * R * 4;                            // of each group's rows: A; E; 2^(25 - E) as a product;
    int *exps = reinterpret_cast<int *>(p); p += 2 * R * 4;
    float2 *units = reinterpret_cast<float2 *>(p); p += 2 * R * 8;
    float2 *changes = reinterpret_cast<float2 *>(p); p += 2 * R * 8;                       // what l and what is summed of O change by
    float *over = reinterpret_cast<float *>(p); p += R * (D == 64 ? 128 : D) * 4;
    float *coefs = reinterpret_cast<float *>(p); p += 2 * (FAN + 3) * MAX_ROWS * 4;         // joining: what a part counts for
    unsigned *cum = reinterpret_cast<unsigned *>(p);
    const uint32_t bar = ptx::smem_u32(control), ring_at = ptx::smem_u32(smem), q_at = ptx::smem_u32(qs), p_at = ptx::smem_u32(ps);
    const uint32_t K_FULL = bar, V_FULL = bar + 64u, K_EMPTY = bar + 128u, V_EMPTY = bar + 192u, S_FULL = bar + 256u, S_EMPTY = bar + 272u, P_FULL = bar + 288u,
                   P_EMPTY = bar + 304u, Q_FULL = bar + 320u, Q_EMPTY = bar + 336u, OVER = bar + 352u, v_ring = ring_at + (uint32_t)a.k_stages * S::STAGE;
    __shared__ unsigned wsum[THREADS / 32], last_flags[2], tmem_slot;
    __shared__ int fresh[2], least_e[2];                                // a tile's weights begin new sums in O; the least E of a group's rows
    __shared__ Work works[WORKS];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        for (int s = 0; s < S::MAX_STAGES; s++) { ptx::mbar_init(K_FULL + 8 * s, 1); ptx::mbar_init(V_FULL + 8 * s, 1); ptx::mbar_init(K_EMPTY + 8 * s, 1); ptx::mbar_init(V_EMPTY + 8 * s, 1); }
        for (int s = 0; s < 2; s++) {
            ptx::mbar_init(S_FULL + 8 * s, 1);
            ptx::mbar_init(S_EMPTY + 8 * s, 4);
            ptx::mbar_init(P_FULL + 8 * s, 4);
            ptx::mbar_init(P_EMPTY + 8 * s, 1);
            ptx::mbar_init(Q_FULL + 8 * s, 1);
            ptx::mbar_init(Q_EMPTY + 8 * s, 9);
            ptx::mbar_init(OVER + 8 * s, 4);
        }
        ptx::mbar_fence_init();
        ptx::tma_prefetch_desc(&map_k);
        ptx::tma_prefetch_desc(&map_v);
    }
    // columns behind the rows' (and rows that a segment does not have) are sums of zeros
    for (int i = tid; i < (2 * S::QB + 2 * S::PB) / 16; i += THREADS) reinterpret_cast<uint4 *>(qs)[i] = make_uint4(0, 0, 0, 0);
    pdl_wait();
    pdl_launch_dependents();
    // units in front of each request
    unsigned carry = 0;
    for (int base = 0; base < a.R; base += THREADS) {
        const int r = base + tid;
        unsigned v = 0;
        if (r < a.R) { const Request x = request(a, r, R); v = (unsigned)x.groups * (unsigned)a.Hkv * (unsigned)(x.tiles + START); }
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
    const unsigned U = carry, P = min(gridDim.x, U), cta = blockIdx.x;            // equal ranges
    const auto bound = [&](unsigned i) { return (unsigned)((unsigned long long)i * U / P); };
    const auto cta_of = [&](unsigned u) { return (unsigned)(((unsigned long long)(u + 1) * P - 1) / U); };
    if (cta >= P) return;
    const unsigned u0 = bound(cta), u1 = bound(cta + 1);
    if (warp == 10) {
        ptx::tmem_alloc(ptx::smem_u32(&tmem_slot), 512);
        ptx::tmem_relinquish();
    }
    ptx::fence_proxy_async_smem();
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::tc_fence_after_sync();
    const uint32_t tmem = tmem_slot, o_cols = tmem + 2 * N;
    const int bshift = 31 - __clz(a.block), tokens = min(a.block, TK), tshift = 31 - __clz(tokens), pieces = TK / tokens;
    const float inf = __int_as_float(0x7f800000);
    bool ok = true;
    const auto give_up = [&](unsigned code) { if (lane == 0) dev_set_error(ERR_WAIT | code); ok = false; };

    if (warp == 8 || warp == 9) {
        // ---- copies: lane = one piece (a block, or the part of it that lies in a tile); a batch is 32 pieces; this warp brings K or V -----------------
        const bool is_k = warp == 8;
        const CUtensorMap *map = is_k ? &map_k : &map_v;
        const uint32_t full0 = is_k ? K_FULL : V_FULL, empty0 = is_k ? K_EMPTY : V_EMPTY, ring = is_k ? ring_at : v_ring;
        const int stages = is_k ? a.k_stages : a.v_stages;
        Walk walk(a, cum, u0, u1, R);
        Segment s;
        int stage = 0, used = 0, t_next = 0;
        uint32_t phase = 0;
        bool more = walk.next(s);
        const int per_batch = 32 / pieces, mine_t = lane / pieces, pc = lane - mine_t * pieces;
        struct Batch { int tiles, row; float ks, vs; bool mine, inner; } b;       // inner: every row sees all keys of the tile
        int phys = 0, h = 0, tok = 0;
        const auto look_up = [&]() {                               // the table entry of this lane's piece of the next batch
            b.tiles = 0; b.mine = false;
            if (!more) return;
            b.tiles = min(per_batch, s.tiles - t_next);
            const int first = (s.x.lo / TK + s.tile + t_next + mine_t) * TK + pc * tokens;
            b.mine = mine_t < b.tiles && first < s.x.seq && first + tokens > s.x.lo;
            const int key0 = first - pc * tokens, pos0 = s.x.seq - s.x.n;
            b.inner = mine_t < b.tiles && (s.x.n == 1 || (key0 + TK <= (a.causal ? pos0 + 1 : s.x.seq) && (a.window == 0 || key0 > s.x.seq - 1 - a.window)));
            if (b.mine) phys = a.table[(size_t)s.r * a.width + (first >> bshift)];
            tok = first & (a.block - 1);
            h = s.h;
            t_next += b.tiles;
            if (t_next == s.tiles) { more = walk.next(s); t_next = 0; }
        };
        const auto resolve = [&]() {                               // its scales and its place in the pool
            b.ks = 0.f; b.vs = 1.f;
            if (!b.mine) return;
            if (phys < 0 || phys >= a.num_blocks) { dev_set_error(kv::ERR_BLOCK_ID); phys = 0; }
            const size_t unit = (size_t)phys * a.Hkv + h;
            if (is_k) { b.ks = a.ks[unit]; b.vs = a.vs[unit]; }
            b.row = (int)((unit * a.block + tok) / (is_k ? 1 : L::V_TOKENS));
        };
        look_up();
        resolve();
        while (b.tiles > 0 && ok) {
            const Batch now = b;
            look_up();
            float most = 0.f;
            if (is_k) {                                            // of tiles that all rows see whole: their largest exponent in the batch; of others, that of all
                const int e = now.mine ? exponent_of(now.vs) : LEAST, ahead = __reduce_max_sync(0xffffffffu, now.inner ? e : LEAST), any = __reduce_max_sync(0xffffffffu, e);
                most = now.inner ? (float)ahead : (float)any + 0.5f;   // (a half: it bounds the rows' own)
            }
            for (int t = 0; t < now.tiles; t++) {
                if (used >= stages && !wait_idle(empty0 + 8 * stage, phase ^ 1u)) { give_up(is_k ? 1u : 2u); break; }
                const bool in = mine_t == t, here = in && now.mine;
                if (is_k && in) {
                    // the slot's last reader, the scores of tile used - SLOTS: this stage was free only after S of tile used - stages, and that came after them
                    scales[(used & (S::SLOTS - 1)) * S::SCALES + pc] = make_float4(now.ks, now.vs, most, now.vs >= 0.f ? now.vs * 0.f : __int_as_float(0x7FC00000));
                }
                const unsigned count = __popc(__ballot_sync(0xffffffffu, here));
                __syncwarp();                                      // the scales are there before the arrival
                if (lane == 0) ptx::mbar_arrive_expect_tx(full0 + 8 * stage, count * (unsigned)(tokens * D));
                if (here) {
                    const uint32_t at = ring + (uint32_t)stage * S::STAGE + (uint32_t)(pc * tokens * (D == 256 ? 128 : D));
#pragma unroll
                    for (int pl = 0; pl < L::PLANES; pl++) ptx::tma_load_2d(at + pl * L::PLANE_BYTES, map, pl * 128, now.row, full0 + 8 * stage);
                }
                used++;
                if (++stage == stages) { stage = 0; phase ^= 1u; }
            }
            resolve();
        }
        if (!ok) for (int i = 0; i < 64; i++) __nanosleep(50000);    // copies in flight end before the CTA's shared memory is another's
    } else if (warp == 11) {
        // ---- queries: the next pair's, while the others are at one --------------------------------------------------------------------------
        // The code is kept short: an SM comes here cold, and sixteen rows unrolled took 11 us to fetch.
        constexpr int LPR = D == 64 ? 16 : 32, RPW = 32 / LPR, PER = D == 256 ? 2 : 1;         // lanes to a row, rows at a time, words of four of a lane
        constexpr int TURNS = R / RPW < 4 ? R / RPW : 4, BATCH = TURNS * RPW;                  // rows whose loads are in flight together
        Walk walk(a, cum, u0, u1, R);
        Segment s = {};
        const int sub = lane / LPR, col = lane % LPR;
        for (int k = 0;; k++) {
            const bool more = walk.next(s);
            const int rows = more ? min(R, s.x.n * a.G - s.rg * R) : 0;
            // lane = row
            const int rho = s.rg * R + lane, query = more ? rho / a.G : 0, pos = s.x.seq - s.x.n + query;
            const long long from = (long long)(s.x.q0 + query) * a.ldq + (long long)(s.h * a.G + rho - query * a.G) * D;
            float4 v[TURNS][PER];
            const auto fetch = [&](int r0, float4 (&v)[TURNS][PER]) {
#pragma unroll
                for (int i = 0; i < TURNS; i++) {
                    const int r = r0 + i * RPW + sub;
                    const T *src = static_cast<const T *>(a.q) + __shfl_sync(0xffffffffu, from, r);
#pragma unroll
                    for (int e = 0; e < PER; e++) {
                        v[i][e] = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (r < rows) v[i][e] = load4(src + 4 * (col + 32 * e));
                    }
                }
            };
            fetch(0, v);
            if (k >= 2 && !wait_idle(Q_EMPTY + 8 * (k & 1), (k / 2 - 1) & 1)) give_up(3u);
            if (!ok) break;
            if (lane == 0) {
                Work &w = works[k % WORKS];
                w.tiles = more ? s.tiles : 0;
                if (more) {
                    const int q0 = s.x.seq - s.x.n + s.rg * R / a.G, q1 = s.x.seq - s.x.n + min(s.rg * R + R - 1, s.x.n * a.G - 1) / a.G;
                    w.min_hi = a.causal ? min(q0, s.x.seq - 1) : s.x.seq - 1; w.max_lo = first_seen(q1, a.window);
                    w.tile0 = s.x.lo / TK + s.tile; w.n = s.x.n; w.q0 = s.x.q0; w.rg = s.rg; w.h = s.h;
                    w.first = s.tile == 0; w.pair0 = s.pair0; w.pair_tiles = s.pair_tiles;
                }
            }
            if (more) {
                unsigned char *to = qs + (k & 1) * S::QB;
#pragma unroll 1
                for (int r0 = 0; r0 < R && (r0 < rows || k < 2); r0 += BATCH) {  // (rows of an earlier segment: what they give is not read)
                    float4 next[TURNS][PER];
                    if (R > BATCH) fetch(r0 + BATCH, next);
                    uint32_t mine = 0;                                           // lane = row: bits of its largest magnitude
#pragma unroll
                    for (int i = 0; i < TURNS; i++) {
                        uint32_t most = 0;
#pragma unroll
                        for (int e = 0; e < PER; e++)
                            most = max(max(most, max(__float_as_uint(v[i][e].x) & 0x7FFFFFFFu, __float_as_uint(v[i][e].y) & 0x7FFFFFFFu)),
                                       max(__float_as_uint(v[i][e].z) & 0x7FFFFFFFu, __float_as_uint(v[i][e].w) & 0x7FFFFFFFu));
                        if constexpr (LPR == 32) {
                            most = __reduce_max_sync(0xffffffffu, most);
                            if (lane == r0 + i) mine = most;
                        } else {
#pragma unroll
                            for (int o = LPR / 2; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
                            const uint32_t other = __shfl_xor_sync(0xffffffffu, most, 16);
                            if (lane >> 1 == (r0 >> 1) + i) mine = (lane & 1) == sub ? most : other;
                        }
                    }
                    // the row in units of its last digit: amax becomes 127 * 256^2; by a power of two first, so that neither factor leaves fp32
                    const float amax = __uint_as_float(mine), bad = mine >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : 0.f;     // digits cannot tell infinities
                    const float p2 = row_factor(amax), f = amax > 0.f ? 127.f * 65536.f / (amax * p2) : 1.f;
                    if (lane >= r0 && lane < r0 + BATCH)
                        rec[(k & 1) * R + lane] = make_float4(a.scale * (CAP ? 1.f / a.softcap : LOG2E) / f / p2 + bad, -inf,
                                                              __int_as_float(a.causal ? min(pos, s.x.seq - 1) : s.x.seq - 1),
                                                              __int_as_float(first_seen(pos, a.window)));
#pragma unroll
                    for (int i = 0; i < TURNS; i++) {
                        const int r = r0 + i * RPW + sub;
                        const float g2 = __shfl_sync(0xffffffffu, p2, r), g1 = __shfl_sync(0xffffffffu, f, r);
#pragma unroll
                        for (int e = 0; e < PER; e++) {
                            const float y[4] = {v[i][e].x, v[i][e].y, v[i][e].z, v[i][e].w};
                            uint32_t w[4];
#pragma unroll
                            for (int m = 0; m < 4; m++) w[m] = (uint32_t)(__float2int_rn(y[m] * g2 * g1) + 0x8080) ^ 0x8080u;     // signed digits in bytes 2, 1, 0
                            const int d = 4 * col;                               // of plane e
#pragma unroll
                            for (int g = 0; g < 3; g++) {
                                const int n = 3 * r + g;
                                const uint32_t sel = g == 0 ? 0x0062u : g == 1 ? 0x0051u : 0x0040u;
                                const uint32_t word = __byte_perm(__byte_perm(w[0], w[1], sel), __byte_perm(w[2], w[3], sel), 0x5410);
                                const int at = D == 64 ? n * 64 + (((d >> 4) ^ ((n >> 1) & 3)) << 4) + (d & 15) : e * N * 128 + n * 128 + (((d >> 4) ^ (n & 7)) << 4) + (d & 15);
                                *reinterpret_cast<uint32_t *>(to + at) = word;
                            }
                        }
                    }
                    if (R > BATCH)
#pragma unroll
                        for (int i = 0; i < TURNS; i++)
#pragma unroll
                            for (int e = 0; e < PER; e++) v[i][e] = next[i][e];
                }
                ptx::fence_proxy_async_smem();
            }
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(Q_FULL + 8 * (k & 1));
            if (!more) break;
        }
    } else if (warp == 10) {
        // ---- products: S of the next tile and PV of the oldest, each as soon as what it needs is there.  S runs up to two tiles ahead, also into the
        // next pair; it must not be waited for before PV, because the next pair's queries may wait for the end of the one before. ------------------
        const uint32_t lead = elected();
        constexpr uint32_t id_s = idesc_s8(N, 0), id_o = idesc_s8(D == 64 ? 2 * NP : NP, 1);
        int st = 0, pst = 0, nth = 0, left = 0;                      // stages; pair, its tiles that are left
        uint32_t ph = 0, pph = 0;
        unsigned j = 0, i = 0;                                       // tiles whose S, whose PV has been issued
        bool end = false;
        const auto there = [&](uint32_t b, uint32_t parity) { return __all_sync(0xffffffffu, test_one(b, parity)) != 0; };
        long long since = clock64();
        while (!end || i < j) {
            bool did = false;
            if (!end && left == 0 && there(Q_FULL + 8 * (nth & 1), (nth >> 1) & 1)) {
                left = works[nth % WORKS].tiles;
                end = left == 0;
                did = true;
            }
            if (left > 0 && there(K_FULL + 8 * st, ph) && (j < 2 || there(S_EMPTY + 8 * (j & 1), ((j >> 1) - 1) & 1))) {
                ptx::tc_fence_after_sync();
                const uint32_t buf = j & 1, kb = ring_at + st * S::STAGE, qb = q_at + (nth & 1) * S::QB;
#pragma unroll
                for (int k = 0; k < D / 32; k++) {
                    const uint64_t kd = D == 64 ? desc_k<64>(kb) + (uint64_t)(2 * k) : desc_k<128>(kb + (k >> 2) * L::PLANE_BYTES) + (uint64_t)(2 * (k & 3));
                    const uint64_t qd = D == 64 ? desc_k<64>(qb) + (uint64_t)(2 * k) : desc_k<128>(qb + (k >> 2) * N * 128) + (uint64_t)(2 * (k & 3));
                    umma_s8(lead, tmem + buf * N, kd, qd, id_s, k > 0);
                }
                umma_commit(lead, S_FULL + 8 * buf);
                if (S::EARLY) umma_commit(lead, K_EMPTY + 8 * st);
                if (--left == 0) { umma_commit(lead, Q_EMPTY + 8 * (nth & 1)); nth++; }
                if (++st == a.k_stages) { st = 0; ph ^= 1u; }
                j++;
                did = true;
            }
            if (i < j && there(P_FULL + 8 * (i & 1), (i >> 1) & 1) && there(V_FULL + 8 * pst, pph)) {
                ptx::tc_fence_after_sync();
                const uint32_t buf = i & 1, begin = fresh[buf] != 0, vb = v_ring + pst * S::STAGE, pb = p_at + buf * S::PB;
#pragma unroll
                for (int pl = 0; pl < DP; pl++)
#pragma unroll
                    for (int k = 0; k < (D == 64 ? 2 : 4); k++)
                        umma_s8(lead, o_cols + buf * S::OC + pl * NP, desc_mn(vb + pl * L::PLANE_BYTES + k * 32 * 128), desc_p<S::P_ROW>(pb + k * 32 * S::P_ROW), id_o, k > 0 || !begin);
                if (!S::EARLY) umma_commit(lead, K_EMPTY + 8 * pst);            // (as many stages as V)
                umma_commit(lead, V_EMPTY + 8 * pst);
                umma_commit(lead, P_EMPTY + 8 * buf);
                if (++pst == a.v_stages) { pst = 0; pph ^= 1u; }
                i++;
                did = true;
            }
            const long long now = clock64();
            if (did) since = now;
            else if (__any_sync(0xffffffffu, now - since > (1ll << 28))) { give_up(4u); break; }
        }
        if (!ok) for (int n = 0; n < 64; n++) __nanosleep(50000);
    } else {
        // ---- thread = key: scores to weights; thread = dim: O.  This group's tiles are every second one --------------------------------------------
        const uint32_t group = warp >> 2, lanes = (uint32_t)(warp & 3) << 21;
        const int gt = tid & 127, gw = warp & 3, parity = D == 64 ? gt >> 6 : 0;
        float *red = reds + group * 4 * R;
        unsigned j = 0, before = 0;                                                 // tiles so far; this group's last one + 1
        // what is the same for all threads of a row is in registers for few rows, for many in shared memory
        constexpr bool HELD = R <= 8;
        constexpr int STEP = R < 8 ? R : 8;                                          // rows whose scores are in registers at a time
        float l[R], acc[DP][R], facs[HELD ? R : 1], As[HELD ? R : 1];
        float *ref = refs + group * R;
        int *exp_of = exps + group * R;
        float2 *unit = units + group * R, *change = changes + group * R;
        const float4 *rc = rec;
        const auto fac = [&](int r) { if constexpr (HELD) return facs[r]; else return rc[r].x; };
        const auto A = [&](int r) { if constexpr (HELD) return As[r]; else return ref[r]; };
        const auto sync = [&]() { asm volatile("bar.sync %0, 128;" ::"r"(1 + group) : "memory"); };
        // Is it so for any of the 128 threads?  A wait that ran out for one warp is everybody's to know: they leave together.
        const auto vote = [&](bool mine) {
            int any;
            asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, %2, 128, p;\n\tselp.s32 %0, 1, 0, q;\n\t}"
                         : "=r"(any) : "r"((int)mine), "r"(1 + group) : "memory");
            return any != 0;
        };
        // O of the tiles since it was last read, in units of 2^(A + E - 25)
        const auto read_o = [&]() {
            const uint32_t i = before - 1;                                         // the last tile whose PV is in it
            if (ok && !wait_warp(P_EMPTY + 8 * group, (i >> 1) & 1)) give_up(9u);
            ptx::tc_fence_after_sync();
#pragma unroll
            for (int pl = 0; pl < DP; pl++)
#pragma unroll
                for (int r0 = 0; r0 < R; r0 += 4) {
                    uint32_t v[16];
                    columns_load(o_cols + group * S::OC + lanes + pl * NP + parity * NP + 4 * r0, v);
                    columns_arrived(v);
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        acc[pl][r0 + r] += fmaf((float)(int)v[4 * r + 3], 16777216.f, fmaf((float)(int)v[4 * r + 2], 65536.f, fmaf((float)(int)v[4 * r + 1], 256.f, (float)(int)v[4 * r])));
                }
            ptx::tc_fence_before_sync();
        };
        for (int nth = 0;; nth++) {
            if (ok && !wait_warp(Q_FULL + 8 * (nth & 1), (nth >> 1) & 1)) give_up(10u);
            if (vote(!ok)) break;
            const Work w = works[nth % WORKS];
            if (w.tiles == 0) break;
            const int row0 = w.rg * R, rows = min(R, w.n * a.G - row0);
            rc = rec + (nth & 1) * R;
            bool since = false;                                                     // O holds tiles of this segment that have not been read
            int held = 0;
            bool begun = false;                                                     // A and E are this segment's
            float least = 0.f;                                                      // the least E of a row
#pragma unroll
            for (int r = 0; r < R; r++) {
                l[r] = 0.f;
                if constexpr (HELD) { facs[r] = rc[r].x; As[r] = NONE; }
#pragma unroll
                for (int pl = 0; pl < DP; pl++) acc[pl][r] = 0.f;
            }
            for (int t = 0; t < w.tiles; t++, j++) {
                if ((j & 1) != group) continue;
                const uint32_t buf = group;
                const int key = (w.tile0 + t) * TK + gt;
                if (ok && !wait_warp(S_FULL + 8 * buf, (j >> 1) & 1)) give_up(11u);
                ptx::tc_fence_after_sync();
                const float4 sc = scales[(j & (S::SLOTS - 1)) * S::SCALES + (gt >> tshift)];
                // rows that the segment does not have go along: they are not read
                float y[R];                                                        // log2 of exp(s)
                const bool grows = !begun || sc.z > least;
                bool again = grows || held >= FLUSH;
#pragma unroll
                for (int r0 = 0; r0 < R; r0 += STEP) {
                    uint32_t v[3 * STEP];
                    columns_load(tmem + lanes + buf * N + 3 * r0, v);
                    columns_arrived(v);
#pragma unroll
                    for (int r = 0; r < STEP; r++) {
                        // |sum| <= 128 * 127 * 256 < 2^22: to fp32 by the bits of 1.5 * 2^23, which is quicker than a conversion
                        const auto whole = [](uint32_t n) { return __uint_as_float(n + 0x4B400000u) - 12582912.f; };
                        const float s = fmaf(whole(v[3 * r]), 65536.f, fmaf(whole(v[3 * r + 1]), 256.f, whole(v[3 * r + 2])));
                        y[r0 + r] = fmaf(s, fac(r0 + r) * sc.x, sc.w);
                    }
                }
                ptx::tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(S_EMPTY + 8 * buf);
                if constexpr (CAP) {
#pragma unroll
                    for (int r = 0; r < R; r++) y[r] = capped(y[r], a.softcap, 0.f);
                }
                if (key - gt + TK - 1 > w.min_hi || key - gt < w.max_lo) {
#pragma unroll
                    for (int r = 0; r < R; r++)
                        if (key > __float_as_int(rc[r].z) || key < __float_as_int(rc[r].w)) y[r] = -inf;
                }
#pragma unroll
                for (int r = 0; r < R; r++) again = again || y[r] > A(r) + LIMIT;
                if (vote(again || !ok)) {
                    if (vote(!ok)) { ok = false; break; }
                    // a weight would be too large, or a scale is: A moves to the row's largest weight, E to the largest scale of the blocks that it sees of.  A
                    // thread has a row: this is code that few tiles come to, so it is kept short.
#pragma unroll
                    for (int r = 0; r < R; r++) {
                        const float m = warp_max(y[r]);
                        if (lane == 0) red[gw * R + r] = m;
                    }
                    if (since) read_o();
                    sync();
                    if (gw == 0) {
                        int E = LEAST;
                        if (gt < R) {
                            const float was = begun ? ref[gt] : NONE, now = fmaxf(was, floorf(fmaxf(fmaxf(red[gt], red[R + gt]), fmaxf(red[2 * R + gt], red[3 * R + gt]))));
                            const int hi = __float_as_int(rc[gt].z), lo = __float_as_int(rc[gt].w), E0 = begun ? exp_of[gt] : LEAST;
                            const bool each = sc.z != floorf(sc.z);                 // rows that may not see all blocks
                            E = each || !grows ? E0 : max(E0, (int)sc.z);
#pragma unroll 1
                            for (int i = 0, k = key - gt; i < pieces && each && grows; i++, k += tokens)
                                if (k <= hi && k + tokens > lo) E = max(E, exponent_of(scales[(j & (S::SLOTS - 1)) * S::SCALES + i].y));
                            ref[gt] = now;
                            exp_of[gt] = E;
                            unit[gt] = pow2_parts((int)TOP - E);
                            change[gt] = make_float2(ex2(was - now), ex2(was - now) * ex2((float)(E0 - E)));
                        }
                        const int least_of = __reduce_min_sync(0xffffffffu, gt < rows ? E : 0x7fffffff);
                        if (gt == 0) least_e[group] = least_of;
                    }
                    sync();
#pragma unroll
                    for (int r = 0; r < R; r++) {
                        const float2 by = change[r];
                        if constexpr (HELD) As[r] = ref[r];
                        l[r] *= by.x;
#pragma unroll
                        for (int pl = 0; pl < DP; pl++) acc[pl][r] *= by.y;
                    }
                    least = (float)least_e[group];
                    begun = true;
                    since = false;
                    held = 0;
                }
                if (j >= 2 && ok && !wait_warp(P_EMPTY + 8 * buf, ((j >> 1) - 1) & 1)) give_up(13u);
                if (gt == 0) fresh[buf] = !since;
                since = true;
                before = j + 1;
                held++;
                // a row of P is a token's (dim 64: a pair's), its digits from the lowest
                constexpr int SWZ = S::P_ROW == 128 ? 7 : S::P_ROW == 64 ? 3 : S::P_ROW == 32 ? 1 : 0, PER128 = S::P_ROW == 128 ? 0 : S::P_ROW == 64 ? 1 : 2;
                const int prow = D == 64 ? gt >> 1 : gt, piece = D == 64 ? (gt & 1) * (NP / 16) : 0, turn = (prow >> PER128) & SWZ;
                const uint32_t to = p_at + buf * S::PB + prow * S::P_ROW;
#pragma unroll
                for (int r0 = 0; r0 < R; r0 += 4) {
                    uint32_t n[4];
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const float weight = ex2(y[r0 + r] - A(r0 + r));                           // a masked score is -inf: 0
                        const float2 by = unit[r0 + r];                                            // (no product in this order leaves fp32 before the last does)
                        l[r0 + r] += weight;
                        n[r] = (__float2uint_rn(weight * by.x * sc.y * by.y) + 0x808080u) ^ 0x808080u;
                    }
                    sts128(to + (((piece + r0 / 4) ^ turn) << 4), n[0], n[1], n[2], n[3]);
                }
                ptx::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(P_FULL + 8 * buf);
            }
            if (vote(!ok)) break;
            // ---- the pair's rows, or the partial sums of a part of it, out -------------------------------------------------------------------------
            if (since) read_o();
            const bool hands_over = (nth & 1) != (int)group;
#pragma unroll
            for (int r = 0; r < R; r++) {
                float sum = l[r];
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                if (lane == 0) red[gw * R + r] = sum;
            }
            sync();
#pragma unroll
            for (int r = 0; r < R; r++) l[r] = (red[r] + red[R + r]) + (red[2 * R + r] + red[3 * R + r]);
            sync();                                                                 // red has been read
            if (lane == 0) ptx::mbar_arrive(Q_EMPTY + 8 * (nth & 1));
            // dim 64: the odd tokens' threads too have a part of each element.  The group that takes over here was the one that handed over before, so
            // nobody reads the buffer any more.
            if (hands_over) {
#pragma unroll
                for (int r = 0; r < R; r++) {
#pragma unroll
                    for (int pl = 0; pl < DP; pl++) over[r * (D == 64 ? 128 : D) + pl * 128 + gt] = acc[pl][r];
                    if (gt == 0) over_ml[r] = make_float4(begun ? A(r) : NONE, (float)(begun ? exp_of[r] : LEAST), l[r], 0.f);
                }
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(OVER + 8 * (nth & 1));
                continue;
            }
            if (ok && !wait_warp(OVER + 8 * (nth & 1), (nth >> 1) & 1)) give_up(14u);
            float2 tops[R];                                                          // A, E
#pragma unroll
            for (int r = 0; r < R; r++) {
                const float4 x = over_ml[r];
                const float2 mine = begun ? make_float2(A(r), (float)exp_of[r]) : make_float2(NONE, (float)LEAST), top = make_float2(fmaxf(mine.x, x.x), fmaxf(mine.y, x.y));
                float f = ex2(mine.x - top.x), g = ex2(x.x - top.x);
                l[r] = l[r] * f + x.z * g;
                f *= ex2(mine.y - top.y);
                g *= ex2(x.y - top.y);
                tops[r] = top;
#pragma unroll
                for (int pl = 0; pl < DP; pl++) acc[pl][r] = acc[pl][r] * f + over[r * (D == 64 ? 128 : D) + pl * 128 + gt] * g;
            }
            if constexpr (D == 64) {                                                 // the two parities' sums
                sync();
#pragma unroll
                for (int r = 0; r < R; r++)
                    if (parity == 1) over[r * 128 + gt] = acc[0][r];
                sync();
#pragma unroll
                for (int r = 0; r < R; r++)
                    if (parity == 0) acc[0][r] += over[r * 128 + 64 + gt];
            }
            const bool writes = D != 64 || gt < 64;
            if (w.tiles != w.pair_tiles) {
                // ---- the CTAs that share the pair meet: FAN neighbours first, then the groups; the last to come joins, in the order of the ranges ------------
                const auto leave = [&](float4 *pml, float *pv, size_t slot) {
                    if (writes)
#pragma unroll
                        for (int r = 0; r < R; r++)
                            if (r < rows) {
#pragma unroll
                                for (int pl = 0; pl < DP; pl++) pv[(slot * MAX_ROWS + r) * D + pl * 128 + gt] = acc[pl][r];
                                if (gt == 0) pml[slot * MAX_ROWS + r] = make_float4(tops[r].x, tops[r].y, l[r], 0.f);
                            }
                };
                const unsigned c0 = cta_of((unsigned)w.pair0), c1 = cta_of((unsigned)(w.pair0 + w.pair_tiles - 1)), groups = (c1 - c0) / FAN + 1;
                const auto slot_of = [&](unsigned k) { return 2 * k + (k == c0 ? 1 : 0); };
                const auto last_of = [&](unsigned *counter, unsigned n) {      // has everybody written?  What was written before is visible then.
                    __threadfence();
                    sync();
                    if (gt == 0) {
                        const unsigned seen = atomicAdd(counter, 1u);
                        last_flags[group] = seen == n - 1;
                        if (seen == n - 1) *counter = 0u;                      // as the next call expects it
                    }
                    sync();
                    const bool last = last_flags[group];
                    if (last) __threadfence();
                    return last;
                };
                float *coef = coefs + group * (FAN + 3) * MAX_ROWS;            // [part][row], then the rows' A, E and sums
                const auto join = [&](const float4 *pml, const float *pv, unsigned first, unsigned step, unsigned n) {
                    constexpr int AT_ONCE = 32 / (R * DP) > 0 ? 32 / (R * DP) : 1;
                    float o[AT_ONCE][DP][R];
                    const auto fetch = [&](unsigned i0) {
#pragma unroll
                        for (int i = 0; i < AT_ONCE; i++)
#pragma unroll
                            for (int r = 0; r < R; r++)
#pragma unroll
                                for (int pl = 0; pl < DP; pl++) {
                                    o[i][pl][r] = 0.f;
                                    if (i0 + i < n && r < rows && writes) o[i][pl][r] = __ldcg(pv + ((size_t)slot_of(first + (i0 + i) * step) * MAX_ROWS + r) * D + pl * 128 + gt);
                                }
                    };
                    fetch(0);
                    {                                                          // eight threads to a row, two parts each: what each part counts for
                        const int r = gt >> 3, i0 = gt & 7;
                        float4 x[2];
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            x[i] = make_float4(NONE, (float)LEAST, 0.f, 0.f);
                            if (r < rows && i0 + 8 * i < (int)n) x[i] = __ldcg(pml + (size_t)slot_of(first + (i0 + 8 * i) * step) * MAX_ROWS + r);
                        }
                        float top_a = fmaxf(x[0].x, x[1].x), top_e = fmaxf(x[0].y, x[1].y), sum = 0.f;
#pragma unroll
                        for (int k = 4; k > 0; k >>= 1) {
                            top_a = fmaxf(top_a, __shfl_xor_sync(0xffffffffu, top_a, k));
                            top_e = fmaxf(top_e, __shfl_xor_sync(0xffffffffu, top_e, k));
                        }
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            const float f = ex2(x[i].x - top_a);
                            sum += x[i].z * f;
                            coef[(i0 + 8 * i) * MAX_ROWS + r] = f * ex2(x[i].y - top_e);
                        }
#pragma unroll
                        for (int k = 4; k > 0; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
                        if (i0 == 0) { coef[FAN * MAX_ROWS + r] = top_a; coef[(FAN + 1) * MAX_ROWS + r] = top_e; coef[(FAN + 2) * MAX_ROWS + r] = sum; }
                    }
                    sync();
#pragma unroll
                    for (int r = 0; r < R; r++) {
                        tops[r] = make_float2(coef[FAN * MAX_ROWS + r], coef[(FAN + 1) * MAX_ROWS + r]);
                        l[r] = coef[(FAN + 2) * MAX_ROWS + r];
#pragma unroll
                        for (int pl = 0; pl < DP; pl++) acc[pl][r] = 0.f;
                    }
#pragma unroll 1
                    for (unsigned i0 = 0;;) {
#pragma unroll
                        for (int i = 0; i < AT_ONCE; i++)
                            if (i0 + i < n)
#pragma unroll
                                for (int r = 0; r < R; r++)
#pragma unroll
                                    for (int pl = 0; pl < DP; pl++) acc[pl][r] = fmaf(o[i][pl][r], coef[(i0 + i) * MAX_ROWS + r], acc[pl][r]);
                        i0 += AT_ONCE;
                        if (i0 >= n) break;
                        fetch(i0);
                    }
                };
                leave(a.part_ml, a.part, 2 * cta + (w.first ? 1 : 0));
                const unsigned g0 = c0 + (cta - c0) / FAN * FAN, in_group = min((unsigned)FAN, c1 - g0 + 1);
                if (!last_of(a.count + slot_of(g0), in_group)) continue;
                join(a.part_ml, a.part, g0, 1, in_group);
                if (groups > 1) {
                    leave(a.part2_ml, a.part2, slot_of(g0));
                    if (!last_of(a.count2 + slot_of(c0), groups)) continue;
                    join(a.part2_ml, a.part2, c0, FAN, groups);
                }
            }
            if (!writes) continue;
#pragma unroll
            for (int r = 0; r < R; r++)
                if (r < rows) {
                    const int rho = row0 + r, query = rho / a.G, head = w.h * a.G + rho - query * a.G;
                    const float inv = l[r] > 0.f ? 1.f / l[r] : (l[r] == 0.f ? 0.f : l[r]);          // nothing seen: zeros
                    const float2 back = pow2_parts((int)(tops[r].y - TOP));
#pragma unroll
                    for (int pl = 0; pl < DP; pl++)
                        static_cast<T *>(a.out)[(long long)(w.q0 + query) * a.ldo + (long long)head * D + pl * 128 + gt] = out_round(T(), l[r] == 0.f ? 0.f : acc[pl][r] * inv * back.x * back.y);
                    if (a.lse && gt == 0) a.lse[(size_t)(w.q0 + query) * a.Hq + head] = l[r] > 0.f ? (tops[r].x + log2f(l[r])) * LN2 : (l[r] == 0.f ? -inf : l[r]);
                }
        }
    }
    __syncthreads();
    ptx::tc_fence_after_sync();
    if (warp == 10) ptx::tmem_dealloc(tmem, 512);
}

// ---- host ---------------------------------------------------------------------------------------------------------------------------
struct Call {
    Args a;
    const int8_t *k, *v;
    int dtype, dim;
};

// Workspace: the arrival counts, then the partial results of two ends of each CTA's range and of the groups of CTAs.
inline size_t ends() { return (size_t)sm_count() * 2; }
inline size_t count_bytes() { return (2 * ends() * 4 + 255) & ~(size_t)255; }
inline size_t workspace_bytes(int dim) { return count_bytes() + 2 * ends() * MAX_ROWS * (16 + (size_t)dim * 4); }
inline void lay_out(Args &a, void *workspace, int dim) {
    unsigned char *p = static_cast<unsigned char *>(workspace);
    a.count = reinterpret_cast<unsigned *>(p);
    a.count2 = a.count + ends();
    a.part_ml = reinterpret_cast<float4 *>(p + count_bytes());
    a.part2_ml = a.part_ml + ends() * MAX_ROWS;
    a.part = reinterpret_cast<float *>(a.part2_ml + ends() * MAX_ROWS);
    a.part2 = a.part + ends() * MAX_ROWS * dim;
}

template <typename T, int D, int R, bool CAP>
inline int launch_t(const Call &c, int rows, cudaStream_t st) {
    using S = Shape<D, R>;
    auto kern = attention_q8_kernel<T, D, R, CAP>;
    const uint64_t tokens = (uint64_t)c.a.num_blocks * c.a.Hkv * c.a.block;
    const uint32_t box = (uint32_t)(c.a.block < TK ? c.a.block : TK);
    CUtensorMap mk, mv;
    int rc = tmap_cached(&mk, c.k, D, tokens, D == 64 ? 64 : 128, box, D == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_128B);
    if (rc == W4A8_OK)
        rc = tmap_cached(&mv, c.v, D == 64 ? 128 : D, D == 64 ? tokens / 2 : tokens, 128, D == 64 ? box / 2 : box, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_128B);
    if (rc != W4A8_OK) return rc;
    // units are counted in 31 bits: so many requests as full tables of them fit, the others in further launches
    const double units = (double)c.a.Hkv * ((rows + R - 1) / R) * ((double)c.a.width * c.a.block / TK + 1 + START);
    const int most = units * MAX_R < 2e9 ? MAX_R : (int)(2e9 / units);
    if (most < 1) return fail(W4A8_ERR_UNSUPPORTED, "attention_q8: %.0f key tiles of a request", units);
    for (int r0 = 0; r0 < c.a.R; r0 += most) {
        Args a = c.a;
        a.R = c.a.R - r0 < most ? c.a.R - r0 : most;
        a.cu_q += r0;
        a.seq_len += r0;
        a.table += (size_t)r0 * a.width;
        const int stages = S::stages(a.R);                          // at most 2 * MAX_STAGES: neither side has more than MAX_STAGES
        a.k_stages = stages / 2;
        a.v_stages = S::EARLY ? stages - a.k_stages : a.k_stages;
        const size_t smem = (size_t)S::fixed_bytes(a.R) + (size_t)(a.k_stages + a.v_stages) * S::STAGE;
        static PerDevice<size_t> configured_dev;
        size_t &configured = configured_dev.get();
        if (smem > configured) {
            cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
            if (e != cudaSuccess) return cuda_fail(e, "attention_q8 smem opt-in");
            configured = smem;
        }
        cudaError_t e = launch_pdl(kern, dim3(sm_count()), dim3(THREADS), smem, st, mk, mv, a);
        if (e != cudaSuccess) return cuda_fail(e, "attention_q8 launch");
    }
    return launch_status("attention_q8");
}

// The narrowest kernel that takes `rows` (queries x heads of a group of the request with most of them) at once.
template <typename T, int D, bool CAP>
inline int launch_d(const Call &c, int rows, cudaStream_t st) {
    if (rows <= 4) return launch_t<T, D, 4, CAP>(c, rows, st);
    if (rows <= 8) return launch_t<T, D, 8, CAP>(c, rows, st);
    return launch_t<T, D, 16, CAP>(c, rows, st);
}

inline int launch(const Call &c, int rows, cudaStream_t st) {
    return kv::by_type(c.dtype, c.dim, [&](auto t, auto d) {
        using T = decltype(t);
        constexpr int D = decltype(d)::value;
        return c.a.softcap > 0.f ? launch_d<T, D, true>(c, rows, st) : launch_d<T, D, false>(c, rows, st);
    });
}

}  // namespace attn
}  // namespace w4a8
