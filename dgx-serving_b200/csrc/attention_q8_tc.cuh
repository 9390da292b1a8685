// Attention of many queries a request (prompts) over the 8-bit paged KV cache on the tcgen05 tensor cores.
//
// Same formula as attention_q8.cuh.  What bounds it: 4 * dim operations for every (query row, key) pair on the tensor cores, and one
// exponential for each pair on the special function units, which at dim 128 take as long.
//  - A CTA takes 256 rows (queries x heads of a group, dim 256: 128) of one kv head as tiles of 128, and walks over the keys in tiles of 128
//    (dim 256: 64).  S = Q K^T and O += P V are tcgen05.mma kind::f16 with fp32 accumulators in tensor memory: S of both row tiles, in whose
//    columns the weights P are then written as fp16, and O of both: 512 columns.  While the warps of one row tile turn its S into P, the
//    tensor core works on the other's.
//  - The cache's codes come in by bulk copies along the block table, four warps turn them into fp16 (exact) in the operands' layout, rows of
//    64 elements with the 128-byte swizzle: K is then K-major, V the same bytes read as MN-major, so neither is transposed.
//  - A thread has one row: maximum, sum and rescaling need no exchange.  The weight that enters the product, exp(s - B) * vs, takes its
//    block's scale in the exponent: x = exp2(f s + log2 vs - B), one multiply-add and one exp2; the sum divides it out again once per block
//    and row.  B is such that the largest x was in [2^7, 2^9) when B was chosen; it moves, and O in tensor memory is rescaled, only when an x would
//    pass 2^15.  (The whole numbers in log2 vs decide that; what is left of them is below 2.)
//  - That holds while scales are between 2^-40 and 2^40.  From the first tile on with one that is not (zero, say), the sum has a reference of its
//    own, A, and a block's x are taken back from B to A by powers of two, or, where they are less than 2^-60 of what B stands for, are the sum's alone.
//    Both ways give the same bits where both can, so a row's result does not depend on scales that it does not see.
//  - fp32 rows enter as two fp16 terms each, Q and P: twice the products, 22 bits.
// One prompt of 4096 tokens, 32 heads of 128 over 8, causal: 201 us, 684 TFLOP/s of the 1633 that a large product reaches.  A step of two row
// tiles and 128 keys took about 4600 cycles, at 206 us, where its products take 2100 and its exponentials 2050: the row's warps, two on a scheduler, are in
// the way, with the maximum (850), the wait for the scores (1450) and the weights (2500).  Steps of 64 keys with two buffers of scores for each row
// tile hid the wait, and had every step's fixed costs twice: 240 us.
#pragma once
#include "attention_q8.cuh"

namespace w4a8 {
namespace attn_tc {

using attn::LOG2E;
using attn::LN2;
using attn::ex2;
using attn::lg2;
using attn::capped;
using attn::elected;
using attn::umma_commit;
using attn::wait_one;
using attn::wait_warp;
using attn::h2_bits;
using attn::sts128;
using attn::NONE;
constexpr unsigned ERR_WAIT = 0xB00u;
constexpr int THREADS = 512;                   // warps 0-3, 4-7: rows of tile 0, 1; 8-11: codes to fp16; 12: copies; 13: products
constexpr int MAX_R = 2048;
constexpr int SCALE_SLOTS = 4;
enum { TILE_PLAIN, TILE_CAPPED, TILE_FAR };    // what a tile's scores need
constexpr int LONG_KEYS = 32768;               // keys of an item beyond which 16-bit rows' sums leave the tensor core with every tile, as fp32 rows' do
constexpr int ORDINARY = 40;                   // exponents of ordinary scales, either way
constexpr float DEAD = -60.f;                  // log2 of a block's largest weight, in what B stands for, below which it is nothing to the products

// A block's scales as the rows take them: ks; the whole number in log2 vs; the rest of it, in [0, 1); 1 / vs.  Once a scale is not ordinary, the last is
// -2^-rest, without the whole number; not a number if vs is none.  0 is 2^-inf.
__device__ __forceinline__ float4 scale_entry(float ks, float vs, bool far) {
    const float e = vs == 0.f ? -__int_as_float(0x7f800000) : (float)attn::exponent_of(vs);
    const uint32_t b = __float_as_uint(vs < 0x1p-100f ? vs * 0x1p64f : vs);
    const float rest = vs == 0.f ? 0.f : lg2(__uint_as_float((b & 0x7FFFFFu) | 0x3F800000u)), back = ex2(-rest);
    return make_float4(ks, e, rest, !far ? back * attn::pow2(-(int)e) : vs < __int_as_float(0x7f800000) && vs >= 0.f ? -back : __int_as_float(0x7FC00000));
}

template <typename T, int D> struct Shape {
    static constexpr bool SPLIT = std::is_same<T, float>::value;
    static constexpr int KT = D == 256 ? 64 : 128, NT = D == 256 ? 1 : 2, TERMS = SPLIT ? 2 : 1;
    static constexpr int ST = SPLIT && D >= 128 ? 1 : 2;                    // fp16 stages of K and of V
    static constexpr int QT = 128 * D * 2, KV = KT * D * 2, RAW = KT * D;    // bytes: one term of a row tile; a stage; its codes
    static constexpr int OFF_KV = NT * TERMS * QT, OFF_RAW = OFF_KV + 2 * ST * KV, OFF_SCALE = OFF_RAW + 2 * RAW, OFF_BAR = OFF_SCALE + SCALE_SLOTS * 8 * 16;
    static constexpr int SMEM = OFF_BAR + 256 + 1024;
    static constexpr int S_COLS = KT, O_COL = 2 * KT;                        // TMEM: two S buffers, then O of each row tile
    static_assert(O_COL + NT * D <= 512 && SMEM <= 227 * 1024, "shape");
};

enum { RAW_FULL = 0, RAW_EMPTY = 2, K_FULL = 4, K_EMPTY = 6, V_FULL = 8, V_EMPTY = 10, S_FULL = 12, P_FULL = 14, PV_DONE = 16, O_FULL = 17, BARS = 19 };

// D[tmem] (+)= A[tmem] B[smem]; A: 128 lanes, two fp16 a column.  B: N x 16 as the descriptor says.  The whole warp comes here and the elected
// lane issues: addresses and descriptors then stay in uniform registers (inside a branch of one lane an instruction took 120 cycles to issue).
__device__ __forceinline__ void umma_f16_ts(uint32_t lead, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(lead) : "memory");
}
__device__ __forceinline__ void umma_f16_ss(uint32_t lead, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(lead) : "memory");
}
// fp32 accumulators (bits [4,6) = 1), fp16 A and B; bit 16: B is MN-major; N >> 3 in [17,23), M >> 4 in [24,29).
__host__ __device__ constexpr uint32_t idesc_f16(int N, int b_mn) { return (1u << 4) | ((uint32_t)b_mn << 16) | ((uint32_t)(N >> 3) << 17) | (8u << 24); }
// MN-major operand, 128-byte swizzle: 64 elements of a row (one k) in 128 bytes, 8 rows 1024 bytes, the next 64 elements `mn_stride` on.
__device__ __forceinline__ uint64_t desc_mn_sw128(uint32_t addr, uint32_t mn_stride) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(mn_stride >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, "
                 "%21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
                 ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
                 "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
                 "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ float4 lds_f4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
    return v;
}
// Bytes (lo: 0 and 1, hi: 2 and 3) of a word of codes + 128 as two fp16 numbers, minus the 128 again: 0x6400 | u is 1024 + u.
template <int SEL>
__device__ __forceinline__ uint32_t codes_f16(uint32_t u) {
    const uint32_t w = __byte_perm(u, 0x64646464u, SEL);
    return h2_bits(__hsub2(*reinterpret_cast<const __half2 *>(&w), __half2half2(__ushort_as_half(0x6480))));   // 1152
}
// Four bytes of codes as two packed pairs of fp16.
__device__ __forceinline__ void widen(uint32_t w, uint32_t &a, uint32_t &b) {
    w ^= 0x80808080u;
    a = codes_f16<0x4140>(w);
    b = codes_f16<0x4342>(w);
}

__device__ __forceinline__ uint64_t pack2u(uint32_t a, uint32_t b) { uint64_t r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(a), "r"(b)); return r; }
__device__ __forceinline__ uint64_t pack2(float a, float b) { return pack2u(__float_as_uint(a), __float_as_uint(b)); }
__device__ __forceinline__ void unpack2(uint64_t x, float &a, float &b) {
    uint32_t u, v;
    asm("mov.b64 {%0, %1}, %2;" : "=r"(u), "=r"(v) : "l"(x));
    a = __uint_as_float(u); b = __uint_as_float(v);
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) { uint64_t r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
__device__ __forceinline__ uint64_t mul2f(uint64_t a, uint64_t b) { uint64_t r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ uint64_t add2f(uint64_t a, uint64_t b) { uint64_t r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }

// Both passes over a tile's scores are loops over 32 columns whose code stays in the instruction cache nearest to the scheduler: written out
// over 128 columns a warp waited for instructions a tenth of the time.  The next 16 columns are on their way while 16 are worked on.
struct RowMask { int key0, hi, lo; };
template <int N> __device__ __forceinline__ void tmem_arrived(uint32_t (&r)[N]) {   // the loads before this are complete; r is not read earlier
#pragma unroll
    for (int e = 0; e < N; e += 16)
        asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(r[e]), "+r"(r[e + 1]), "+r"(r[e + 2]), "+r"(r[e + 3]), "+r"(r[e + 4]), "+r"(r[e + 5]), "+r"(r[e + 6]),
                     "+r"(r[e + 7]), "+r"(r[e + 8]), "+r"(r[e + 9]), "+r"(r[e + 10]), "+r"(r[e + 11]), "+r"(r[e + 12]), "+r"(r[e + 13]), "+r"(r[e + 14]),
                     "+r"(r[e + 15]) :: "memory");
}
// The columns of a tile in steps of N, the next step's on their way while one is worked on: step(registers, first column).
template <int KT, int N, class Step>
__device__ __forceinline__ void columns(uint32_t at, Step &&step) {
    static_assert(KT % (2 * N) == 0, "two steps a trip");
    uint32_t v[2][N];
    ptx::tmem_ld(at, v[0]);
#pragma unroll 1
    for (int c = 0; c < KT; c += 2 * N) {
        tmem_arrived(v[0]);
        ptx::tmem_ld(at + c + N, v[1]);
        step(v[0], c);
        tmem_arrived(v[1]);
        if (c + 2 * N < KT) ptx::tmem_ld(at + c + 2 * N, v[0]);
        step(v[1], c + N);
    }
}
// log2 of the row's largest exp(s) * 2^e, e the whole number in log2 vs; FAR: and of its largest exp(s).
template <int KT, int N, bool EDGE, bool FAR>
__device__ __forceinline__ float2 top_of(uint32_t s_at, uint32_t sc, float fac, float cap, const RowMask &k) {
    const float inf = __int_as_float(0x7f800000);
    float top = -inf, top_z = -inf;
    columns<KT, N>(s_at, [&](uint32_t (&r)[N], int c) {
        float4 k4[N / 16];                                                   // scale_entry
#pragma unroll
        for (int u = 0; u < N / 16; u++) k4[u] = lds_f4(sc + c + 16 * u);
        if (EDGE) {
#pragma unroll
            for (int e = 0; e < N; e++)
                if (k.key0 + c + e > k.hi || k.key0 + c + e < k.lo) r[e] = 0xff800000u;
        }
#pragma unroll
        for (int u = 0; u < N / 16; u++) {
            float m[4];
#pragma unroll
            for (int e = 0; e < 4; e++)
                m[e] = fmaxf(fmaxf(__uint_as_float(r[16 * u + e]), __uint_as_float(r[16 * u + 4 + e])), fmaxf(__uint_as_float(r[16 * u + 8 + e]), __uint_as_float(r[16 * u + 12 + e])));
            const float mm = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])), f = fac * k4[u].x;
            if (FAR) {
                top_z = fmaxf(top_z, cap > 0.f ? (mm == -inf ? -inf : capped(mm * f, cap, 0.f)) : mm * f);
            }
            top = fmaxf(top, cap > 0.f ? (mm == -inf ? -inf : capped(mm * f, cap, k4[u].y)) : fmaf(mm, f, k4[u].y));
        }
    });
    return make_float2(top, top_z);
}
// The weights in place of the scores: 16 columns of scores become 8 of fp16 pairs (fp32 rows: and 8 of what they round off).  l += their sum.
template <int KT, int N, bool SPLIT, bool EDGE, bool CAP, bool FAR>
__device__ __forceinline__ void weights(uint32_t s_at, uint32_t sc, float fac, float cap, float A, float B, const RowMask &k, float &l) {
    columns<KT, N>(s_at, [&](const uint32_t (&r)[N], int c) {
        float4 k4[N / 16];
        float p[N];
#pragma unroll
        for (int u = 0; u < N / 16; u++) k4[u] = lds_f4(sc + c + 16 * u);
        float back[N / 16];                                                  // what brings the block's x to the sum's units
        bool dead[N / 16];
#pragma unroll
        for (int u = 0; u < N / 16; u++) {
            const float f = fac * k4[u].x;
            float add = (k4[u].y - B) + k4[u].z;
            back[u] = k4[u].w;
            dead[u] = false;
            if (FAR) {
                const float d = B - A;
                dead[u] = k4[u].y - d < DEAD;
                if (dead[u]) add = -A;
                add += 0.f * k4[u].w;                                        // (not a number where the scale is none)
                back[u] = dead[u] ? 1.f : -k4[u].w * ex2(d - k4[u].y);
            }
            if (CAP) {
                float x[16], most = 0.f;
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    x[e] = __uint_as_float(r[16 * u + e]) * f;
                    most = fmaxf(most, fabsf(x[e]));
                }
                if (FAR && !(cap > 0.f)) {
#pragma unroll
                    for (int e = 0; e < 16; e++) p[16 * u + e] = ex2(fmaf(__uint_as_float(r[16 * u + e]), f, add));
                } else if (__any_sync(0xffffffffu, most > attn::SMALL_X)) {
#pragma unroll
                    for (int e = 0; e < 16; e++) p[16 * u + e] = ex2(capped(x[e], cap, add));
                } else {                                                     // the same as capped, two at a time
                    const uint64_t c3 = pack2(attn::TANH3, attn::TANH3), c5 = pack2(attn::TANH5, attn::TANH5), c7 = pack2(attn::TANH7, attn::TANH7), c9 = pack2(attn::TANH9, attn::TANH9),
                                   by = pack2(cap * LOG2E, cap * LOG2E), a2 = pack2(add, add);
#pragma unroll
                    for (int e = 0; e < 16; e += 2) {
                        const uint64_t v = pack2(x[e], x[e + 1]), w = mul2f(v, v);
                        const uint64_t t = fma2(mul2f(v, w), fma2(fma2(fma2(c9, w, c7), w, c5), w, c3), v);
                        float y0, y1;
                        unpack2(fma2(by, t, a2), y0, y1);
                        p[16 * u + e] = ex2(y0);
                        p[16 * u + e + 1] = ex2(y1);
                    }
                }
            } else {
                const uint64_t f2 = pack2(f, f), a2 = pack2(add, add);
#pragma unroll
                for (int e = 16 * u; e < 16 * u + 16; e += 2) {
                    unpack2(fma2(pack2u(r[e], r[e + 1]), f2, a2), p[e], p[e + 1]);
                    p[e] = ex2(p[e]);
                    p[e + 1] = ex2(p[e + 1]);
                }
            }
        }
        if (EDGE) {
#pragma unroll
            for (int e = 0; e < N; e++)
                if (k.key0 + c + e > k.hi || k.key0 + c + e < k.lo) p[e] = 0.f;
        }
#pragma unroll
        for (int u = 0; u < N / 16; u++) {
            const float *q = p + 16 * u;
            uint64_t sum[4];
#pragma unroll
            for (int e = 0; e < 4; e++) sum[e] = add2f(pack2(q[4 * e], q[4 * e + 1]), pack2(q[4 * e + 2], q[4 * e + 3]));
            float s0, s1;
            unpack2(add2f(add2f(sum[0], sum[1]), add2f(sum[2], sum[3])), s0, s1);
            if (!FAR || s0 + s1 != 0.f) l = fmaf(s0 + s1, back[u], l);       // (a block that is all masked may have a scale that is not a number)
            uint32_t ph[8], pl[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const __half2 b = __floats2half2_rn(q[2 * e], q[2 * e + 1]);
                ph[e] = h2_bits(b);
                if (SPLIT) {
                    const float2 back = __half22float2(b);
                    pl[e] = h2_bits(__floats2half2_rn(q[2 * e] - back.x, q[2 * e + 1] - back.y));
                }
            }
            if (FAR && dead[u])
#pragma unroll
                for (int e = 0; e < 8; e++) ph[e] = pl[e] = 0u;
            tmem_st8(s_at + c + 16 * u, ph);
            if (SPLIT) tmem_st8(s_at + c + 16 * u + 8, pl);
        }
    });
}
// 32 rows of Q by one warp: whole rows at a time, a row's largest magnitude by shuffles, its scaled fp16 terms into the operand's layout (row 0 of
// the 32 at `dst`; the second term `term` bytes on).  fac[row]: what brings a score back, without a.scale.  Rows from `there` on are zeros.
template <typename T, int D, bool SPLIT, class RowAt>
__device__ __forceinline__ void rows_in(uint32_t dst, uint32_t term, float *fac, bool minus, int there, int lane, RowAt &&row_at) {
    constexpr int N = kv::Row<T>::N, LPR = D / N, PER = LPR > 32 ? LPR / 32 : 1, RPW = LPR >= 32 ? 1 : 32 / LPR, BATCH = 32 / RPW < 16 / PER ? 32 / RPW : 16 / PER;
    const int sub = LPR >= 32 ? 0 : lane / LPR, col = lane & (LPR >= 32 ? 31 : LPR - 1);
#pragma unroll 1
    for (int r0 = 0; r0 < 32; r0 += RPW * BATCH) {
        uint4 raw[BATCH][PER];
#pragma unroll
        for (int b = 0; b < BATCH; b++) {
            const int r = r0 + b * RPW + sub;
#pragma unroll
            for (int q = 0; q < PER; q++)
                raw[b][q] = r < there ? *reinterpret_cast<const uint4 *>(row_at(r) + (col + 32 * q) * N) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int b = 0; b < BATCH; b++) {
            const int r = r0 + b * RPW + sub;
            float x[PER][N];
            uint32_t most = 0;                                                 // bits of the largest magnitude
#pragma unroll
            for (int q = 0; q < PER; q++) {
                kv::Row<T>::unpack(raw[b][q], x[q]);
#pragma unroll
                for (int e = 0; e < N; e++) most = max(most, __float_as_uint(x[q][e]) & 0x7FFFFFFFu);
            }
            if constexpr (LPR >= 32) most = __reduce_max_sync(0xffffffffu, most);
            else {
#pragma unroll
                for (int o = LPR / 2; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
            }
            float f = attn::row_factor(__uint_as_float(most));
            if (col == 0) fac[r] = 1.f / f;
            if (minus) f = -f;
#pragma unroll
            for (int q = 0; q < PER; q++) {
                const int at = (col + 32 * q) * N, chunk = at >> 3;            // of 8 elements
                const uint32_t to = dst + r * 128 + (chunk >> 3) * (128 * 128) + (((chunk & 7) ^ (r & 7)) << 4) + (at & 7) * 2;
                uint32_t h[N / 2], lo[N / 2];
#pragma unroll
                for (int e = 0; e < N / 2; e++) {
                    const float u = x[q][2 * e] * f, v = x[q][2 * e + 1] * f;
                    const __half2 t = __floats2half2_rn(u, v);
                    const float2 back = __half22float2(t);
                    h[e] = h2_bits(t);
                    lo[e] = h2_bits(__floats2half2_rn(u - back.x, v - back.y));
                }
                if constexpr (N == 8) sts128(to, h[0], h[1], h[2], h[3]);
                else {
                    asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(to), "r"(h[0]), "r"(h[1]) : "memory");
                    if (SPLIT) asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(to + term), "r"(lo[0]), "r"(lo[1]) : "memory");
                }
            }
        }
    }
}

// The block is launched with 128 registers a thread; the rows' two warpgroups take 200, the others keep 56: 2 * 128 * (200 + 56) = 512 * 128.
template <int N> __device__ __forceinline__ void raise_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void lower_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }


// N columns of a thread's row, times inv (a product of two), into the staging rows of its warp: `bytes` a row, piece c of 16 bytes at c ^ (row & 7).
template <int N, typename T> __device__ __forceinline__ void stage(uint32_t at, int row, int col, const float (&y)[N], float2 inv) {
    constexpr int E = 16 / sizeof(T);
#pragma unroll
    for (int e = 0; e < N; e += E) {
        float x[E];
#pragma unroll
        for (int i = 0; i < E; i++) x[i] = inv.x == 0.f ? 0.f : y[e + i] * inv.x * inv.y;
        const uint4 w = kv::Row<T>::pack(x);
        sts128(at + ((((col + e) / E) ^ (row & 7)) << 4), w.x, w.y, w.z, w.w);
    }
}
// The staged 32 rows of a warp (the first at `at`, `stride` bytes apart, pieces from `piece0` on) to memory, whole rows at a time; lane = row of `dst`.
template <int N, typename T> __device__ __forceinline__ void rows_out(uint32_t at, uint32_t stride, int piece0, T *dst, int there, int lane) {
    constexpr int PIECES = N * (int)sizeof(T) / 16, ROWS = 32 / PIECES;
    __syncwarp();
#pragma unroll 4
    for (int r0 = 0; r0 < 32; r0 += ROWS) {
        const int r = r0 + lane / PIECES, c = lane % PIECES;
        T *to = reinterpret_cast<T *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(dst), r));
        const uint4 w = lds128(at + r * stride + (((piece0 + c) ^ (r & 7)) << 4));
        if (r < there) *reinterpret_cast<uint4 *>(to + c * (16 / (int)sizeof(T))) = w;
    }
}
// O = O * by + 128 columns of tensor memory.
__device__ __forceinline__ void add_columns(float (&O)[128], uint32_t at, float by) {
#pragma unroll
    for (int c = 0; c < 4; c++) {
        uint32_t o[32];
        ptx::tmem_ld(at + 32 * c, o);
        ptx::tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 32; e++) O[32 * c + e] = fmaf(O[32 * c + e], by, __uint_as_float(o[e]));
    }
}

// The tensor core's sums lose up to a unit in the last place with every sixteen keys, toward zero: 16-bit rows over 131072 keys were off by 7.9e-4, over
// 2^20 by 6.3e-3.  SUMS: they are one tile's, and the rows' sums over the tiles are held in registers (fp32 rows; 16-bit rows over more than LONG_KEYS keys, which
// are LONG's; 32768 lose 1.9e-4, less than fp16's rounding).
template <typename T, int D, bool LONG>
__global__ void __launch_bounds__(THREADS, 1) attention_q8_tc_kernel(const attn::Args a, const int8_t *__restrict__ kc, const int8_t *__restrict__ vc) {
    using S = Shape<T, D>;
    constexpr int KT = S::KT, NT = S::NT, ST = S::ST, TERMS = S::TERMS;
    constexpr bool SPLIT = S::SPLIT, SUMS = SPLIT || LONG;
    constexpr int STEP = SUMS ? 16 : 32;           // columns of scores in work; where the registers do not hold O, more
    constexpr int OWN = D < 128 ? D : 128;         // columns of O that a thread sums itself (SUMS)
    extern __shared__ unsigned char smem_raw[];
    __shared__ unsigned wsum[THREADS / 32];
    __shared__ int item[4];                       // request, kv head, row tile
    __shared__ uint32_t tmem_slot;
    __shared__ float shrinks[2][128];              // the rows' factors; dim 256, fp32 rows: what O is rescaled by, two tiles' worth, then what divides it
    float *const facs = NT == 1 ? shrinks[1] : shrinks[0];
    unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t base = ptx::smem_u32(smem), bars = base + S::OFF_BAR, scales = base + S::OFF_SCALE;
    const auto BAR = [&](int i) { return bars + 8u * i; };
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_wait();
    pdl_launch_dependents();
    // ---- which rows: the blockIdx.x-th item of all requests that have more than `few` rows --------------------------------------------
    if (tid == 0) item[0] = -1;
    {
        unsigned carry = 0;
        __syncthreads();
        for (int r0 = 0; r0 < a.R; r0 += THREADS) {
            const int r = r0 + tid;
            unsigned v = 0;
            if (r < a.R) {
                const int q0 = max(0, min(a.cu_q[r], a.T)), n = max(0, min(a.cu_q[r + 1], a.T) - q0), rows = n * a.G;
                if (rows > a.few) v = (unsigned)((rows + NT * 128 - 1) / (NT * 128)) * (unsigned)a.Hkv;
            }
            unsigned s = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const unsigned t = __shfl_up_sync(0xffffffffu, s, o); if (lane >= o) s += t; }
            if (lane == 31) wsum[warp] = s;
            __syncthreads();
            unsigned front = carry;
            for (int w = 0; w < warp; w++) front += wsum[w];
            const unsigned lo = front + s - v;
            if (v != 0 && blockIdx.x >= lo && blockIdx.x < lo + v) {
                // the request's last rows first: with the causal mask they have the most keys
                const unsigned in = blockIdx.x - lo, tiles = v / (unsigned)a.Hkv;
                item[0] = r;
                item[1] = (int)(in % (unsigned)a.Hkv);
                item[2] = (int)(tiles - 1 - in / (unsigned)a.Hkv);
            }
            for (int w = 0; w < THREADS / 32; w++) carry += wsum[w];
            __syncthreads();
            if (item[0] >= 0) break;
        }
    }
    const int r = item[0];
    if (r < 0) return;
    const attn::Request x = attn::request(a, r, 1);
    const int h = item[1], row0 = item[2] * NT * 128, rows = x.n * a.G;
    const int nt = NT == 2 && row0 + 128 < rows ? 2 : 1;                          // row tiles with rows in them
    const int last_row = min(row0 + NT * 128, rows) - 1;
    const int first_q = row0 / a.G, last_q = last_row / a.G;
    const int lo_all = attn::first_seen(x.seq - x.n + first_q, a.window);
    const int hi_all = a.causal ? x.seq - x.n + last_q + 1 : x.seq;               // keys [lo_all, hi_all) for some row
    const int tile0 = lo_all / KT, n = hi_all > lo_all ? (hi_all + KT - 1) / KT - tile0 : 0;

    if (!SPLIT && (n * KT > LONG_KEYS) != LONG) return;                          // the other kernel's

    if (warp == 13) {
        ptx::tmem_alloc(ptx::smem_u32(&tmem_slot), 512);
        ptx::tmem_relinquish();
    }
    if (tid == 0) {
        constexpr int P_COUNT = SUMS && NT == 1 ? 256 : 128;
        const int counts[BARS] = {1, 1, 4, 4, 4, 4, 1, 1, 4, 4, 1, 1, 1, 1, P_COUNT, P_COUNT, 1, 1, 1};
        for (int i = 0; i < BARS; i++) ptx::mbar_init(BAR(i), counts[i]);
        ptx::mbar_fence_init();
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::tc_fence_after_sync();
    const uint32_t tmem = tmem_slot;
    bool ok = true;

    if (warp < 8 && warp / 4 < nt) {
        // ---- a row tile's warps: thread = row -----------------------------------------------------------------------------------------
        raise_registers<200>();
        const int t = warp >> 2, row = row0 + t * 128 + (tid & 127);
        const int query = min(row, rows - 1) / a.G, head = h * a.G + min(row, rows - 1) % a.G;
        const int at = x.seq - x.n + query;
        const int hi = a.causal ? min(at, x.seq - 1) : x.seq - 1, lo = attn::first_seen(at, a.window);
        const int min_hi = __reduce_min_sync(0xffffffffu, hi), max_lo = __reduce_max_sync(0xffffffffu, lo);
        float fac = 0.f;
        if (n > 0) {
            const int first = row0 + (tid & ~31);                            // of this warp's rows
            rows_in<T, D, SPLIT>(base + t * TERMS * S::QT + (tid & 96) * 128, S::QT, facs + (tid & ~31), a.scale < 0.f, rows - first, lane, [&](int i) {
                const int q = (first + i) / a.G;
                return static_cast<const T *>(a.q) + (long long)(x.q0 + q) * a.ldq + (long long)(h * a.G + first + i - q * a.G) * D;
            });
            __syncwarp();
            fac = fabsf(a.scale) * (a.softcap > 0.f ? 1.f / a.softcap : LOG2E) * facs[tid];
            ptx::fence_proxy_async_smem();
            asm volatile("bar.arrive %0, 160;" ::"r"(1 + t) : "memory");       // the product warp waits for the tile's Q
        }
        const float inf = __int_as_float(0x7f800000);
        const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21);
        const uint32_t o_at = lanes + S::O_COL + t * D;
        // SUMS: O in tensor memory is one tile's
        float O[SUMS ? OWN : 1];
        if constexpr (SUMS) {
#pragma unroll
            for (int e = 0; e < OWN; e++) O[e] = 0.f;
        }
        float A = NONE, B = NONE, l = 0.f, shrink = 1.f;             // A follows B until a tile is far
        const auto take = [&](float by) {                            // O of the tile before, complete in tensor memory, into the registers
            if constexpr (SUMS) {
#pragma unroll
                for (int c = 0; c < OWN / 32; c++) {
                    uint32_t o[32];
                    ptx::tmem_ld(o_at + 32 * c, o);
                    ptx::tmem_ld_wait();
#pragma unroll
                    for (int e = 0; e < 32; e++) O[32 * c + e] = fmaf(O[32 * c + e], by, __uint_as_float(o[e]));
                }
            }
        };
        // One tile's scores to weights.  false, and nothing done, where it is the first with a scale that is not ordinary and `kind` does not know them.
        const auto tile = [&](auto kind, int j) {
            constexpr bool FAR = decltype(kind)::value == TILE_FAR, CAP = decltype(kind)::value == TILE_CAPPED;
            const int buf = NT == 2 ? t : j & 1;
            const uint32_t s_at = lanes + buf * S::S_COLS;
            if (ok && !wait_warp(BAR(S_FULL + buf), (NT == 2 ? j : j >> 1) & 1)) { if (lane == 0) dev_set_error(ERR_WAIT | 1u); ok = false; }
            ptx::tc_fence_after_sync();
            const uint32_t sc = scales + (j & (SCALE_SLOTS - 1)) * 128;
            if (!FAR && !(lds_f4(sc).w > 0.f)) return false;
            const int key0 = (tile0 + j) * KT;
            const bool edge = key0 + KT - 1 > min_hi || key0 < max_lo;
            const auto products_before = [&]() {                     // one S buffer ahead: O is whole when PV of tile j - 1 is done
                if (ok && !wait_warp(BAR(PV_DONE), (j - 1) & 1)) { if (lane == 0) dev_set_error(ERR_WAIT | 2u); ok = false; }
                ptx::tc_fence_after_sync();
            };
            bool waited = NT == 2 || j == 0;                         // two row tiles: S_t of this tile came after PV_t of the one before
            if (SUMS && NT == 2 && j > 0) take(shrink);
            const RowMask mask = {key0, hi, lo};
            float2 top;
            if constexpr (FAR) top = top_of<KT, 16, true, true>(s_at, sc, fac, a.softcap, mask);
            else {
                const float cap = CAP ? a.softcap : 0.f;
                top = edge ? top_of<KT, CAP ? 16 : STEP, true, false>(s_at, sc, fac, cap, mask) : top_of<KT, CAP ? 16 : STEP, false, false>(s_at, sc, fac, cap, mask);
            }
            const bool again = top.x > B + 14.f || (FAR && top.y > A + 60.f);
            shrink = 1.f;
            if (__any_sync(0xffffffffu, again)) {
                const float Bn = top.x > B + 14.f ? floorf(top.x) - 7.f : B, An = !FAR ? Bn : top.y > A + 60.f ? floorf(top.y) : A;
                shrink = ex2(B - Bn);                                // nothing is summed before the first
                l *= ex2(A - An);
                A = An;
                B = Bn;
                if (!SUMS && j > 0) {
                    if (!waited) { products_before(); waited = true; }
#pragma unroll 1
                    for (int c = 0; c < D / 32; c++) {
                        uint32_t o[32];
                        ptx::tmem_ld(o_at + 32 * c, o);
                        ptx::tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * shrink);
                        tmem_st32(o_at + 32 * c, o);
                    }
                }
            }
            float sum = 0.f;                                         // of the tile: one addition for each tile to the row's, not one for sixteen keys
            if constexpr (FAR) weights<KT, 16, SPLIT, true, true, true>(s_at, sc, fac, a.softcap, A, B, mask, sum);
            else if constexpr (CAP) {
                if (edge) weights<KT, 16, SPLIT, true, true, false>(s_at, sc, fac, a.softcap, A, B, mask, sum);
                else weights<KT, 16, SPLIT, false, true, false>(s_at, sc, fac, a.softcap, A, B, mask, sum);
            }
            else if (edge) weights<KT, STEP, SPLIT, true, false, false>(s_at, sc, fac, 0.f, A, B, mask, sum);
            else weights<KT, STEP, SPLIT, false, false, false>(s_at, sc, fac, 0.f, A, B, mask, sum);
            l += sum;
            if (SUMS && NT == 1) {
                if (j > 0) { products_before(); take(shrinks[(j - 1) & 1][tid]); }
                shrinks[j & 1][tid] = shrink;                        // for the other half's warps, who read it before PV of tile j + 1
            } else if (!waited) products_before();                   // every phase is awaited, so none is mistaken for another
            tmem_st_wait();
            ptx::tc_fence_before_sync();
            ptx::mbar_arrive(BAR(P_FULL + buf));
            return true;
        };
        int j = 0;                                                   // loops of their own: a choice in one cost 6 % of a prompt's time, and more with caps
        if (a.softcap > 0.f) while (j < n && tile(std::integral_constant<int, TILE_CAPPED>(), j)) j++;
        else while (j < n && tile(std::integral_constant<int, TILE_PLAIN>(), j)) j++;
        for (; j < n; j++) tile(std::integral_constant<int, TILE_FAR>(), j);
        // ---- the rows out ------------------------------------------------------------------------------------------------------------
        if (n > 0) {
            if (ok && !wait_warp(BAR(O_FULL + t), 0)) { if (lane == 0) dev_set_error(ERR_WAIT | 3u); ok = false; }
            ptx::tc_fence_after_sync();
            take(shrink);
        }
        const float2 unit = attn::pow2_parts((int)fminf(fmaxf(B - A, -250.f), 250.f));
        const float2 inv = make_float2((l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l)) * unit.x, unit.y);
        if (SUMS && NT == 1) {
            asm volatile("bar.sync 4, 256;" ::: "memory");           // the other half has read the last factor
            shrinks[0][tid] = inv.x;
            shrinks[1][tid] = inv.y;
            asm volatile("bar.sync 3, 256;" ::: "memory");
        }
        // through shared memory, where Q was (every product is done): stored by its own thread a row took 16 bytes of each of 32 rows at a time
        T *dst = static_cast<T *>(a.out) + (long long)(x.q0 + query) * a.ldo + (long long)head * D;
        constexpr uint32_t ROW = D * sizeof(T);
        static_assert(sizeof(T) == 2 * TERMS, "a row of the output takes what its terms took");
        const uint32_t rows_at = base + t * TERMS * S::QT + (tid & 96) * ROW, row_at = rows_at + lane * ROW;
        const int there = rows - (row0 + t * 128 + (tid & 96));
        if constexpr (SUMS) {
            stage<OWN, T>(row_at, lane, 0, O, inv);
            rows_out<OWN, T>(rows_at, ROW, 0, dst, there, lane);
        } else {
#pragma unroll 1
            for (int c = 0; c < D / 32; c++) {
                uint32_t o[32];
                float y[32];
#pragma unroll
                for (int e = 0; e < 32; e++) o[e] = 0u;
                if (n > 0) {
                    ptx::tmem_ld(o_at + 32 * c, o);
                    ptx::tmem_ld_wait();
                }
#pragma unroll
                for (int e = 0; e < 32; e++) y[e] = __uint_as_float(o[e]);
                stage<32, T>(row_at, lane, 32 * c, y, inv);
            }
            rows_out<D, T>(rows_at, ROW, 0, dst, there, lane);
        }
        if (a.lse && row < rows) a.lse[(size_t)(x.q0 + query) * a.Hq + head] = l > 0.f ? (A + log2f(l)) * LN2 : (l == 0.f ? -inf : l);
        ptx::tc_fence_before_sync();
    } else if (SUMS && NT == 1 && warp >= 4 && warp < 8) {
        // ---- dim 256, SUMS: the second half of O's columns ----------------------------------------------------------------------------
        raise_registers<200>();
        const int lr = tid & 127, row = row0 + lr, query = min(row, rows - 1) / a.G, head = h * a.G + min(row, rows - 1) % a.G;
        const uint32_t o_at = tmem + ((uint32_t)(warp & 3) << 21) + S::O_COL + 128;
        float O[128];
#pragma unroll
        for (int e = 0; e < 128; e++) O[e] = 0.f;
        for (int j = 0; j < n; j++) {
            if (j > 0) {                                             // the first tile's weights wait for nobody
                if (ok && !wait_warp(BAR(PV_DONE), (j - 1) & 1)) { if (lane == 0) dev_set_error(ERR_WAIT | 13u); ok = false; }
                ptx::tc_fence_after_sync();
                add_columns(O, o_at, shrinks[(j - 1) & 1][lr]);
                ptx::tc_fence_before_sync();
            }
            ptx::mbar_arrive(BAR(P_FULL + (j & 1)));
        }
        if (n > 0) {
            if (ok && !wait_warp(BAR(O_FULL), 0)) { if (lane == 0) dev_set_error(ERR_WAIT | 14u); ok = false; }
            ptx::tc_fence_after_sync();
            add_columns(O, o_at, shrinks[(n - 1) & 1][lr]);
        }
        asm volatile("bar.sync 4, 256;" ::: "memory");
        asm volatile("bar.sync 3, 256;" ::: "memory");
        const uint32_t rows_at = base + (tid & 96) * (D * sizeof(T));
        stage<128, T>(rows_at + lane * (D * sizeof(T)), lane, 128, O, make_float2(shrinks[0][lr], shrinks[1][lr]));
        rows_out<128, T>(rows_at, D * sizeof(T), 128 * (int)sizeof(T) / 16, static_cast<T *>(a.out) + (long long)(x.q0 + query) * a.ldo + (long long)head * D + 128, rows - (row0 + (tid & 96)), lane);
        ptx::tc_fence_before_sync();
    } else if (warp >= 8 && warp < 12) {
        // ---- codes to fp16 -------------------------------------------------------------------------------------------------------------
        lower_registers<56>();
        const uint32_t k8 = lane >> 2, cq = lane & 3, odd4 = D == 64 ? 0 : (k8 & 1) * 4, my_key = (warp - 8) * 8 + k8;
        const uint32_t my_src = my_key * D + 16 * cq, my_dst = my_key * 128, pos0 = ((2 * cq) ^ k8) << 4, pos1 = ((2 * cq + 1) ^ k8) << 4;
        for (int j = 0; j < n; j++) {
            const int st = j % ST;
#pragma unroll
            for (int kv = 0; kv < 2; kv++) {
                const int full = kv ? V_FULL : K_FULL, empty = kv ? V_EMPTY : K_EMPTY;
                if (ok && !wait_warp(BAR(RAW_FULL + kv), j & 1)) { if (lane == 0) dev_set_error(ERR_WAIT | 4u); ok = false; }
                if (ok && j >= ST && !wait_warp(BAR(empty + st), (j / ST - 1) & 1)) { if (lane == 0) dev_set_error(ERR_WAIT | 5u); ok = false; }
                const uint32_t src = base + S::OFF_RAW + kv * S::RAW, dst = base + S::OFF_KV + (2 * st + kv) * S::KV;
                // A warp takes eight tokens and four 16-byte pieces of their codes at a time; odd tokens the other four of eight, so that neither
                // the reads nor the two writes meet a bank twice.
                constexpr int CH = D / 16;
                if (ok)
#pragma unroll
                    for (int k0 = 0; k0 < KT; k0 += 32)
#pragma unroll
                        for (int it = 0; it < CH / 4; it++) {
                            const int flip = D == 64 ? 0 : 4 * (it & 1), off = 8 * (it >> 1);
                            const uint32_t c4 = odd4 ^ flip;                 // 0 or 4
                            const uint4 w = lds128(src + my_src + k0 * D + 16 * (c4 + off));
                            uint32_t f[8];
                            widen(w.x, f[0], f[1]);
                            widen(w.y, f[2], f[3]);
                            widen(w.z, f[4], f[5]);
                            widen(w.w, f[6], f[7]);
                            const uint32_t to = dst + my_dst + k0 * 128 + (c4 >> 2) * (KT * 128) + (off >> 2) * (KT * 128);
                            sts128(to + pos0, f[0], f[1], f[2], f[3]);
                            sts128(to + pos1, f[4], f[5], f[6], f[7]);
                        }
                ptx::fence_proxy_async_smem();
                __syncwarp();
                if (ok && lane == 0) {
                    ptx::mbar_arrive(BAR(RAW_EMPTY + kv));
                    ptx::mbar_arrive(BAR(full + st));
                }
            }
        }
    } else if (warp >= 12) {
        lower_registers<56>();
        if (warp == 12) {
        // ---- copies: lane = one piece of a tile (a block, or the part of it in the tile) --------------------------------------------------
        const int piece = min(a.block, KT), pieces = KT / piece, per = piece / 16, bshift = 31 - __clz(a.block);
        const auto entry = [&](int j) {                             // block id of this lane's piece of tile j; -1: no token that is seen
            const int first = (tile0 + j) * KT + lane * piece;
            if (lane >= pieces || j >= n || first >= hi_all || first + piece <= lo_all) return -1;
            int id = a.table[(size_t)r * a.width + (first >> bshift)];
            if (id < 0 || id >= a.num_blocks) { dev_set_error(kv::ERR_BLOCK_ID); id = 0; }
            return id;
        };
        int id = entry(0);
        float ks = 0.f, vs = 1.f;
        bool far = false;
        const float least = attn::pow2(-ORDINARY), most = attn::pow2(ORDINARY);
        if (id >= 0) { ks = a.ks[(size_t)id * a.Hkv + h]; vs = a.vs[(size_t)id * a.Hkv + h]; }
        for (int j = 0; j < n && ok; j++) {
            const int next = entry(j + 1);
            const unsigned count = __popc(__ballot_sync(0xffffffffu, id >= 0));
            const int first = (tile0 + j) * KT + lane * piece;
            const size_t off = id >= 0 ? (((size_t)id * a.Hkv + h) * a.block + (first & (a.block - 1))) * D : 0;
            if (j > 0 && !wait_warp(BAR(RAW_EMPTY), (j - 1) & 1)) { if (lane == 0) dev_set_error(ERR_WAIT | 6u); ok = false; break; }
            far = far || __any_sync(0xffffffffu, !(vs >= least && vs < most));
            const float4 x = scale_entry(ks, vs, far);
            // the slot's last reader was tile j - 4's rows, done before this K can be awaited (two stages and one tile of codes ahead)
            if (lane < pieces) {
                for (int u = 0; u < per; u++) {
                    const uint32_t to = scales + (j & (SCALE_SLOTS - 1)) * 128 + (lane * per + u) * 16;
                    sts128(to, __float_as_uint(x.x), __float_as_uint(x.y), __float_as_uint(x.z), __float_as_uint(x.w));
                }
            }
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive_expect_tx(BAR(RAW_FULL), count * (unsigned)(piece * D));
            if (id >= 0) bulk_load(base + S::OFF_RAW + lane * piece * D, kc + off, piece * D, BAR(RAW_FULL));
            if (j > 0 && !wait_warp(BAR(RAW_EMPTY + 1), (j - 1) & 1)) { if (lane == 0) dev_set_error(ERR_WAIT | 7u); ok = false; break; }
            if (lane == 0) ptx::mbar_arrive_expect_tx(BAR(RAW_FULL + 1), count * (unsigned)(piece * D));
            __syncwarp();
            if (id >= 0) bulk_load(base + S::OFF_RAW + S::RAW + lane * piece * D, vc + off, piece * D, BAR(RAW_FULL + 1));
            id = next;
            ks = 0.f; vs = 1.f;
            if (id >= 0) { ks = a.ks[(size_t)id * a.Hkv + h]; vs = a.vs[(size_t)id * a.Hkv + h]; }
        }
        if (!ok) for (int i = 0; i < 64; i++) __nanosleep(50000);
    } else if (warp == 13 && n > 0) {
        // ---- products ------------------------------------------------------------------------------------------------------------------
        for (int t = 0; t < nt; t++) asm volatile("bar.sync %0, 160;" ::"r"(1 + t) : "memory");
        const uint32_t lead = elected();
        {
            constexpr uint32_t id_s = idesc_f16(KT, 0), id_o = idesc_f16(D, 1);
            const auto wait = [&](int bar, int parity, unsigned code) {
                if (ok && !wait_warp(BAR(bar), parity & 1)) { if (lane == 0) dev_set_error(ERR_WAIT | code); ok = false; }
                ptx::tc_fence_after_sync();
                return ok;
            };
            const auto scores = [&](int t, int j, int buf) {
                const uint32_t kb = base + S::OFF_KV + 2 * (j % ST) * S::KV;
                uint32_t first = 0;
#pragma unroll
                for (int term = 0; term < TERMS; term++)
#pragma unroll
                    for (int k = 0; k < D / 16; k++) {
                        const uint64_t qd = ptx::umma_desc_k_sw128(base + (t * TERMS + term) * S::QT + (k >> 2) * 128 * 128) + (uint64_t)((k & 3) * 2);
                        const uint64_t kd = ptx::umma_desc_k_sw128(kb + (k >> 2) * KT * 128) + (uint64_t)((k & 3) * 2);
                        umma_f16_ss(lead, tmem + buf * S::S_COLS, qd, kd, id_s, first);
                        first = 1;
                    }
                umma_commit(lead, BAR(S_FULL + buf));
            };
            const auto values = [&](int t, int j, int buf) {
                const uint32_t vb = base + S::OFF_KV + (2 * (j % ST) + 1) * S::KV;
#pragma unroll
                for (int term = 0; term < TERMS; term++)
#pragma unroll
                    for (int k = 0; k < KT / 16; k++)
                        umma_f16_ts(lead, tmem + S::O_COL + t * D, tmem + buf * S::S_COLS + 16 * k + 8 * term,
                                    desc_mn_sw128(vb + k * 16 * 128, KT * 128), id_o, (!SUMS && j > 0) || term > 0 || k > 0);
            };
            wait(K_FULL, 0, 8u);
            if (ok) {
                for (int t = 0; t < nt; t++) scores(t, 0, t);
                umma_commit(lead, BAR(K_EMPTY));
            }
            for (int j = 0; j < n && ok; j++) {
                const int st = j % ST, s1 = (j + 1) % ST;
                if (NT == 1 && j + 1 < n) {
                    if (!wait(K_FULL + s1, (j + 1) / ST, 9u)) break;
                    scores(0, j + 1, (j + 1) & 1);
                    umma_commit(lead, BAR(K_EMPTY + s1));
                }
                for (int t = 0; t < nt; t++) {
                    const int buf = NT == 2 ? t : j & 1;
                    if (t == 0 && !wait(V_FULL + st, j / ST, 10u)) break;
                    if (!wait(P_FULL + buf, NT == 2 ? j : j >> 1, 11u)) break;
                    values(t, j, buf);
                    if (t == nt - 1) umma_commit(lead, BAR(V_EMPTY + st));
                    if (NT == 1) umma_commit(lead, BAR(PV_DONE));
                    if (j == n - 1) umma_commit(lead, BAR(O_FULL + t));
                    if (NT == 2 && j + 1 < n) {
                        if (t == 0 && !wait(K_FULL + s1, (j + 1) / ST, 12u)) break;
                        scores(t, j + 1, t);
                        if (t == nt - 1) umma_commit(lead, BAR(K_EMPTY + s1));
                    }
                }
            }
            if (!ok) for (int i = 0; i < 64; i++) __nanosleep(50000);
        }
        __syncwarp();
        }
    }
    __syncthreads();
    ptx::tc_fence_after_sync();
    if (warp == 13) ptx::tmem_dealloc(tmem, 512);
}

template <typename T, int D, bool LONG>
inline int launch_t(const attn::Call &c, cudaStream_t st) {
    using S = Shape<T, D>;
    auto kern = attention_q8_tc_kernel<T, D, LONG>;
    static PerDevice<bool> configured;
    if (!configured.get()) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
        if (e != cudaSuccess) return cuda_fail(e, "attention_q8_tc smem opt-in");
        configured.get() = true;
    }
    // no more items than full tiles of all rows and a partial one for each request
    const long long rows = (long long)c.a.T * c.a.G, items = (rows / (S::NT * 128) + (c.a.R < c.a.T ? c.a.R : c.a.T)) * c.a.Hkv;
    if (items > 0x7fffffffll) return fail(W4A8_ERR_UNSUPPORTED, "attention_q8: %lld row tiles", items);
    cudaError_t e = launch_pdl(kern, dim3((unsigned)items), dim3(THREADS), S::SMEM, st, c.a, c.k, c.v);
    return e == cudaSuccess ? launch_status("attention_q8_tc") : cuda_fail(e, "attention_q8_tc launch");
}

inline int launch(const attn::Call &c, cudaStream_t st) {
    return kv::by_type(c.dtype, c.dim, [&](auto t, auto d) {
        using T = decltype(t);
        constexpr int D = decltype(d)::value;
        const int rc = launch_t<T, D, false>(c, st);
        if constexpr (!Shape<T, D>::SPLIT)                              // can a request be that long?
            if (rc == W4A8_OK && (long long)c.a.width * c.a.block > LONG_KEYS) return launch_t<T, D, true>(c, st);
        return rc;
    });
}

}  // namespace attn_tc
}  // namespace w4a8
