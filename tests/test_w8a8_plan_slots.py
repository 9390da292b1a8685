"""csrc/gemm_w8a8_plan.cuh on the CPU: where plans are kept, the same shape on several GPUs of one process has a place for each."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dgx-serving_b200", "csrc")

DRIVER = r"""
#include "gemm_w8a8_plan.cuh"
#include <cstdio>
#include <set>
using namespace w4a8::w8a8;
int main() {
    for (int M : {1, 2, 17, 64, 333, 2048, MAX_ROWS})
        for (int N : {1, 300, 4091, 6144, 17408, MAX_ROWS})
            for (int K : {32, 512, 5120, 131040}) {
                std::set<int> slots;
                for (int dev = 0; dev < 16; dev++) {
                    const int s = plan_slot(M, N, K, dev);
                    if (s < 0 || s >= PLAN_SLOTS || !slots.insert(s).second) return printf("M %d N %d K %d dev %d: slot %d\n", M, N, K, dev, s), 1;
                }
            }
    std::set<int> used;                                                     // shapes of a decode loop spread out
    for (int M = 1; M <= 64; M++)
        for (int N : {3840, 4096, 6144, 17408}) used.insert(plan_slot(M, N, 5120, 0));
    return used.size() < 128;
}
"""


def test_a_shape_has_a_place_on_every_gpu(tmp_path):
    src, exe = tmp_path / "slots.cpp", tmp_path / "slots"
    src.write_text(DRIVER)
    r = subprocess.run(["g++", "-O2", "-std=c++17", "-x", "c++", "-I", CSRC, "-o", str(exe), str(src)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout
