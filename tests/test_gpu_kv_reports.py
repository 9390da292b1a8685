"""GPU tests of what the KV cache's kernels report through device_status."""
import numpy as np
import pytest
import torch

from conftest import to_dev
from test_gpu_kv_cache import pool

pytestmark = pytest.mark.gpu


def test_two_errors_are_reported_one_after_the_other(w4a8, cuda):
    """A slot beyond the cache and a wait that nothing ends: neither hides the other."""
    arenas = [w4a8.Arena(4096, r, 2) for r in range(2)]
    try:
        for a in arenas:
            a.connect_pointers([b.base for b in arenas])
        dev = [to_dev(a, cuda) for a in pool(np.random.default_rng(1), 2, 1, 16, 64)]
        x = torch.ones((1, 64), device=cuda)
        arenas[0].wait(7, timeout_us=2000)                                            # nobody published epoch 7
        w4a8.launch_kv_append_q8(x, x, 64, to_dev(np.array([99], np.int32), cuda), 1, w4a8.KVCache.of(*dev))
        texts = []
        for _ in range(2):
            with pytest.raises(w4a8.W4A8Error) as e:
                w4a8.device_status()
            assert e.value.code == w4a8.ERR_DEVICE
            texts.append(str(e.value))
        assert sum("slot" in t for t in texts) == 1 and sum("wait" in t for t in texts) == 1
        w4a8.device_status()
    finally:
        for a in arenas:
            a.close()
