"""csrc/gemm_w8a8_plan.cuh on the CPU, over many sizes: every plan is one that the kernel can run."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dgx-serving_b200", "csrc")

DRIVER = r"""
#include "gemm_w8a8_plan.cuh"
#include <cstdio>
#include <initializer_list>
using namespace w4a8::w8a8;
int main() {
    int bad = 0, rows = 0, kinds[3] = {};
    const Caps whole = {148, {0, 0, 74, 45, 33, 0, 22, 0, 15}}, small = {132, {0, 0, 60, 0, 14, 0, 0, 0, 3}};
    for (const Caps &caps : {whole, small})
        for (int M : {1, 2, 15, 16, 17, 31, 33, 48, 49, 64, 65, 100, 128, 129, 200, 255, 256, 257, 300, 333, 512, 777, 1000, 2048, 5000, 100000, MAX_ROWS})
            for (int N : {1, 5, 63, 64, 65, 127, 128, 129, 255, 300, 1024, 3840, 4091, 6144, 17408, 151936, MAX_ROWS})
                for (int K : {32, 96, 128, 160, 256, 512, 1056, 4096, 5120, 15360, 32768, 131040}) {
                    const Plan p = plan_for(M, N, K, caps);
                    const long tiles = (long)ceil_div(N, p.bw) * ceil_div(M, p.bt);
                    bool ok = p.bt >= 16 && p.bt <= 256 && p.bt % (p.pair ? 32 : 16) == 0 && p.kp >= 1 && stages_for(p) >= 2 && stages_for(p) <= MAX_STAGES && smem_for(p) <= SMEM_MAX;
                    ok = ok && (p.pair ? p.bw == 2 * LANES && p.split == 1 && p.at_once == caps.clusters[2] : p.bw >= 8 && p.bw <= LANES && p.bw % 8 == 0);
                    if (p.split > 1) {                                  // all clusters at once; each CTA has K-tiles; its rows fit a warp's registers, the sums the stages' memory
                        ok = ok && p.split <= SPLIT_MAX && tiles <= caps.clusters[p.split] && ceil_div(K, KT) >= p.split && p.bt <= SPLIT_BT && ceil_div(p.bt, p.split) <= 64;
                        ok = ok && p.bt * LANES * 4 <= stages_for(p) * stage_bytes_for(p);
                    }
                    Plan q = p;
                    if (row_plan(q, M, K)) {                            // a row or two quantized by the product: sixteen rows of the CTA's K beside the stages
                        rows++;
                        ok = ok && M <= ROWS_MAX && q.bt == 16 && !q.pair && row_stages_for(q, K) >= 3 && (q.kp == 2 || q.kp == 1) && row_stages_for(q, K) <= MAX_STAGES && row_smem_for(q, K) <= SMEM_MAX;
                        ok = ok && (ceil_div(K, KT) + q.split - 1) / q.split * 16 * KT <= row_bytes(q, K) && split_receive(q.bt, q.split) % 1024 == 0;
                        ok = ok && (q.split == 1 || q.bt * LANES * 4 <= row_stages_for(q, K) * A_STAGE * q.kp);
                    }
                    kinds[p.pair ? 2 : p.split > 1]++;
                    if (!ok && bad++ < 10) printf("M %d N %d K %d: bw %d bt %d split %d kp %d pair %d\n", M, N, K, p.bw, p.bt, p.split, p.kp, p.pair);
                }
    printf("%d bad, kinds %d %d %d\n", bad, kinds[0], kinds[1], kinds[2]);
    return bad || !kinds[0] || !kinds[1] || !kinds[2] || !rows;
}
"""


def test_every_plan_can_be_run(tmp_path):
    src, exe = tmp_path / "plan.cpp", tmp_path / "plan"
    src.write_text(DRIVER)
    subprocess.run(["g++", "-O2", "-std=c++17", "-x", "c++", "-I", CSRC, "-o", str(exe), str(src)], check=True, capture_output=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout
