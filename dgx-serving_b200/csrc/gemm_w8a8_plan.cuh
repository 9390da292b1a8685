// How an 8-bit product (gemm_w8a8.cuh) is cut into tiles: sizes alone, no CUDA construct, so that the CPU can go through it for all of them.
#pragma once
#include <initializer_list>

namespace w4a8 {
namespace w8a8 {

constexpr int MAX_K = 131040, MAX_ROWS = 0x7fffffff - 1023;
constexpr int LANES = 128, KT = 128;           // channels of an MMA; bytes of K in a row of a swizzled tile
constexpr int A_STAGE = LANES * KT;
constexpr int MAX_STAGES = 12, EPI_WARPS = 8, THREADS = (2 + EPI_WARPS) * 32;
constexpr int SMEM_MAX = 227 * 1024, SMEM_FIXED = 1024 /* alignment */ + 512 /* barriers */;
constexpr int SPLIT_MAX = 8, SPLIT_BT = 128;   // CTAs that share a tile, and the widest tile that they share

// How the outputs are cut: tiles of bw channels and bt rows, split CTAs to a tile.
// pair: two CTAs to a tile, of 256 channels.  at_once: pairs that fit the GPU.
struct Plan { int bw, bt, split, kp, pair, at_once; };
inline int ceil_div(long a, long b) { return (int)((a + b - 1) / b); }

inline int split_receive(int bt, int split) { return split > 1 ? split * ceil_div(bt, split) * LANES * 4 : 0; }
inline int stages_for(const Plan &p) {
    const int n = (SMEM_MAX - SMEM_FIXED - split_receive(p.bt, p.split)) / ((A_STAGE + (p.pair ? p.bt / 2 : p.bt) * KT) * p.kp);
    return n > MAX_STAGES ? MAX_STAGES : n;
}

// What a plan takes, in us: a launch; for each wave of tiles the K-tiles' copies (1.5 ns a row of 128 bytes, both operands'; shared memory fills at 85 bytes a
// ns), MMAs (pairs) or hand-offs (0.12 a K-tile and 0.16 a stage), whichever is most, or the outputs of the tile before; the weights from HBM; and what sums
// between CTAs and pairs cost.  Fitted to 1600 shapes (M 1 to 3000, N 256 to 20000, K 256 to 16384), each timed behind its quantizer with some 30 to
// 150 plans on a B200: the plan that it picks is 2.2 % slower than the best of them on average, 6.5 % at the 90th percentile, 25 % at most.
struct Caps { int sms, clusters[SPLIT_MAX + 1]; };                     // clusters of n CTAs that fit the GPU at once
inline int k_parts(int bt, int split, bool pair) {                     // fewer hand-offs, as long as three stages fit
    if (pair) return bt <= 160 ? 2 : 1;
    return split > 1 ? 2 : bt <= 16 ? 4 : bt <= 128 ? 2 : 1;
}
inline float cost_of(const Plan &p, int M, int N, int K, const Caps &caps) {
    const long tiles = (long)ceil_div(N, p.bw) * ceil_div(M, p.bt);
    const int at_once = p.pair ? caps.clusters[2] : p.split > 1 ? caps.clusters[p.split] : caps.sms;
    // clusters of one wave; of threes the last two that should fit were seen to wait for others (44 and 45 of 45 took 1.2 times as long)
    if (at_once <= 0 || (p.split > 1 && tiles > at_once - (p.split == 3 ? 2 : 0))) return 1e30f;
    const float waves = (float)((tiles + at_once - 1) / at_once), k_tiles = (float)ceil_div(ceil_div(K, KT), p.split);
    const float mma = p.pair ? 0.134f + 1.23e-3f * p.bt : 0.f, fill = 1.5e-3f * (p.pair ? LANES + p.bt / 2 : p.bw + p.bt), hand = 0.124f + 0.156f / p.kp;
    const float per = k_tiles * (mma > fill ? (mma > hand ? mma : hand) : fill > hand ? fill : hand);
    const float out = 0.0123f * p.bt * (p.pair ? 1.39f : 1.f) + 1.19f;
    const float body = (waves - 1.f) * (per > out ? per : out) + per + out, mem = (float)N * (float)K / 16.1e6f;
    return 2.4f + (body > mem ? body + 0.35f * mem : mem + 0.35f * body) + (p.split > 1 ? 0.53f + 0.029f * p.bt : 0.f) + (p.pair ? 0.5f : 0.f);
}
inline Plan plan_for(int M, int N, int K, const Caps &caps) {
    Plan best = {LANES, 256, 1, 1, 0, caps.sms};
    float least = 2e30f;
    const auto try_plan = [&](Plan p) {
        p.kp = k_parts(p.bt, p.split, p.pair != 0);
        if (stages_for(p) < 2) return;
        const float c = cost_of(p, M, N, K, caps);
        p.at_once = p.pair ? caps.clusters[2] : caps.sms;
        if (c < least) { least = c; best = p; }
    };
    const int nkt = ceil_div(K, KT);
    int last = 0;
    for (int widest = 256; widest >= 16; widest -= 16) {               // M in as many parts as this width makes, as even as sixteens allow
        const int bt = ceil_div(ceil_div(M, ceil_div(M, widest)), 16) * 16;
        if (bt == last) continue;
        last = bt;
        for (int bw = 64; bw <= LANES; bw += 32) {
            try_plan({bw, bt, 1, 0, 0, 0});
            for (const int split : {2, 3, 4, 8})
                if (bt <= SPLIT_BT && nkt / split >= 2) try_plan({bw, bt, split, 0, 0, 0});
        }
        try_plan({2 * LANES, ceil_div(bt, 32) * 32, 1, 0, 1, 0});
        if (bt <= 48) break;
    }
    return best;
}
// Where the plan of a shape is kept: the GPU turns the place, so that the same layers on several GPUs do not put one another out.
constexpr int PLAN_SLOTS = 256;
inline int plan_slot(int M, int N, int K, int dev) { return (((unsigned)M * 2654435761u ^ (unsigned)N * 2246822519u ^ (unsigned)K * 3266489917u) + (unsigned)dev * 2654435769u) >> 24; }
inline int stage_bytes_for(const Plan &p) { return (A_STAGE + (p.pair ? p.bt / 2 : p.bt) * KT) * p.kp; }
inline int smem_for(const Plan &p) { return stages_for(p) * stage_bytes_for(p) + SMEM_FIXED + split_receive(p.bt, p.split); }

// Rows that the product quantizes itself stay in shared memory, a CTA's part of K of sixteen rows (the MMA's narrowest), and the stages hold weights alone.
constexpr int ROWS_MAX = 2;
inline int row_bytes(const Plan &p, int K) { return (ceil_div(ceil_div(K, KT), p.split) + (p.split > 1)) * 16 * KT; }
inline int row_stages_for(const Plan &p, int K) {
    const int n = (SMEM_MAX - SMEM_FIXED - 1024 - split_receive(p.bt, p.split) - row_bytes(p, K)) / (A_STAGE * p.kp);
    return n > MAX_STAGES ? MAX_STAGES : n;
}
inline int row_smem_for(const Plan &p, int K) { return row_stages_for(p, K) * A_STAGE * p.kp + SMEM_FIXED + 1024 + split_receive(p.bt, p.split) + row_bytes(p, K); }
// Whether a product of M rows quantizes them itself, and how: a single row wherever it fits beside stages of 96 KB (5120 x 17408 beside 64 KB: 20.1 / 27.0), two of up to 8192 elements, which the threads
// keep between their two looks.  us in a graph, two launches / one, 17408 x 5120 18.5 / 16.8, 8192 x 3840 11.0 / 8.3, 4096 x 4096 8.3 / 6.1, 3840 x 15360 14.4 / 13.8;
// two rows 18.6 / 17.8, 11.1 / 8.5, 8.4 / 7.0, 14.5 / 16.4; three 18.3 / 19.5, 11.2 / 9.4, 8.4 / 8.1, 14.4 / 18.8.
inline bool row_plan(Plan &p, int M, int K) {
    if (M > ROWS_MAX || (M > 1 && K > 8192) || p.pair || p.bt != 16) return false;
    p.kp = 2;
    return row_stages_for(p, K) >= 3;
}

}  // namespace w8a8
}  // namespace w4a8
