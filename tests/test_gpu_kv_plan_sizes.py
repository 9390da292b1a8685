"""Plans whose sums take about as much shared memory as a launch gets without asking for more (48 KB, what the kernel keeps besides included)."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
SIZES = (6143, 6125, 6124, 6144, 16384)


def plan(R):
    import numpy as np
    import torch

    import kv_plain
    from conftest import load_package
    from test_gpu_kv_cache import plan_on_gpu
    kv, new = np.arange(R, dtype=np.int32) % 37, 1 + np.arange(R, dtype=np.int32) % 2
    table = np.full((R, 3), -1, np.int32)
    have = -(-kv // 16)
    at = np.concatenate([[0], np.cumsum(have)])
    for r in range(R):
        table[r, : have[r]] = np.arange(at[r], at[r + 1])
    free = np.arange(at[-1], at[-1] + R // 8, dtype=np.int32)                  # too few for the last requests
    T = int(new.sum())
    want = kv_plain.plan(kv, new, 16, table, free, 0, T)
    got = plan_on_gpu(load_package(), torch.device("cuda:0"), kv, new, 16, table, free, 0, T)
    for k in want:
        assert np.array_equal(got[k], want[k]), (R, k)


def test_sizes_around_48_kb():
    """In a process of its own: a larger plan before these would have asked for them too."""
    r = subprocess.run([sys.executable, os.path.abspath(__file__)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


if __name__ == "__main__":
    for R in SIZES:
        plan(R)
