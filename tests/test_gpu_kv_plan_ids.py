"""Block ids in a plan's table or free list that no slot can be made of: the rows get none, and device_status says so."""
import numpy as np
import pytest

from test_gpu_kv_cache import plan_on_gpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("block", [16, 128])
@pytest.mark.parametrize("bad", [2 ** 31 // 16, 2 ** 31 - 1, -1, -2 ** 31])
@pytest.mark.parametrize("held", [True, False])
def test_ids_whose_slots_do_not_fit(w4a8, cuda, block, bad, held):
    """Such an id times the block's tokens may wrap to a slot of another request."""
    import torch
    table, free = np.array([[bad if held else 1, -1], [2, -1]], np.int32), [3 if held else bad, 4]
    kv, new = [3 if held else block, 5], [2, 2]
    with pytest.raises(w4a8.W4A8Error) as e:
        plan_on_gpu(w4a8, cuda, kv, new, block, table, free, 0, 4)
    assert e.value.code == w4a8.ERR_DEVICE and "block" in str(e.value)
    dev = lambda a: torch.tensor(a, dtype=torch.int32, device=cuda)
    out = [torch.full((n,), -9, dtype=torch.int32, device=cuda) for n in (2, 3, 4, 4, 4)]
    w4a8.kv_plan(dev(kv), dev(new), 2, block, dev(table), 2, dev(free), 2, dev([0]), *out[:4], 4, out[4])
    with pytest.raises(w4a8.W4A8Error):
        w4a8.device_status()
    assert out[2].tolist() == [-1, -1, 2 * block + 5, 2 * block + 6]
