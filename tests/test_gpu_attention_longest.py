"""GPU tests of requests with about 2^31 tokens, of which a window sees the last ones: positions a tile further do not wrap."""
import numpy as np
import pytest
import torch

import kv_plain
from conftest import to_dev

pytestmark = pytest.mark.gpu
LONGEST = 2 ** 31 - 512


@pytest.mark.parametrize("rows", [1, 3, 70])
@pytest.mark.parametrize("D,causal", [(64, 1), (128, 0), (256, 1)])
@pytest.mark.parametrize("seq", [LONGEST, LONGEST - 129, 2 ** 31 - 1])
def test_last_tokens_of_the_longest_requests(w4a8, cuda, rows, D, causal, seq):
    """More than 2^31 - 512 tokens are reported."""
    rng, block, window = np.random.default_rng(D + rows), 128, 50
    k, v = (rng.integers(-127, 128, (4, 1, block, D)).astype(np.int8) for _ in range(2))
    ks, vs = ((rng.random((4, 1)) * 0.01 + 0.01).astype(np.float32) for _ in range(2))
    cache = w4a8.KVCache.of(*(to_dev(a, cuda) for a in (k, v, ks, vs)))
    last = (seq - 1) // block
    table = torch.full((1, 2 ** 24), -1, dtype=torch.int32, device=cuda)
    table[0, last - 3:last + 1] = torch.arange(4, dtype=torch.int32, device=cuda)
    q = rng.standard_normal((rows, 2, D)).astype(np.float32)
    out = torch.zeros((rows, 2, D), device=cuda)
    ws = torch.zeros(w4a8.attention_q8_workspace_bytes(2, cache), dtype=torch.uint8, device=cuda)
    w4a8.launch_attention_q8(to_dev(q, cuda), 2 * D, cache, table, 2 ** 24, to_dev(np.array([0, rows], np.int32), cuda), to_dev(np.array([seq], np.int32), cuda), 1, rows, 2,
                             out, 2 * D, D ** -0.5, "fp32", ws, causal=causal, window=window, max_q=rows)
    if seq > LONGEST:
        with pytest.raises(w4a8.W4A8Error) as e:
            w4a8.device_status()
        assert e.value.code == w4a8.ERR_DEVICE and "2^31" in str(e.value)
        return
    w4a8.device_status()
    held = seq - (last - 3) * block                               # the request as if it began with the four blocks
    kk, vv = ([kv_plain.rows_of(c, s, np.arange(4), held)] for c, s in ((k, ks), (v, vs)))
    o, _, reach = kv_plain.attention(q.astype(np.float64), np.array([0, rows]), [held], kk, vv, D ** -0.5, causal=causal, window=window)
    weight = reach * 2.0 ** -23 * (D / 16 + 8) + 2.0 ** -18         # as in the attention tests
    assert (np.abs(out.cpu().numpy() - o) <= 2 * (weight + 2.0 ** -18) * np.abs(vv[0]).max() + 2.0 ** -23 * np.abs(o)).all()


def test_plan_of_more_tokens_than_a_request_can_have(w4a8, cuda):
    """Such a request is not served, and takes no block from the others."""
    dev = lambda a: torch.tensor(a, dtype=torch.int32, device=cuda)
    table = torch.full((2, 2 ** 24 + 8), -1, dtype=torch.int32, device=cuda)
    table[0, (2 ** 31 - 512) // 128 - 1] = 5
    out = [torch.full((n,), -9, dtype=torch.int32, device=cuda) for n in (2, 3, 4, 4, 4)]
    w4a8.kv_plan(dev([2 ** 31 - 513, 0]), dev([2, 1]), 2, 128, table, 2 ** 24 + 8, dev([7, 8]), 2, dev([0]), *out[:4], 4, out[4])
    w4a8.device_status()
    assert out[0].tolist() == [0, 1] and out[2].tolist() == [-1, -1, 7 * 128, -1] and out[4].tolist() == [1, 1, 1, 1]
    w4a8.kv_plan(dev([2 ** 31 - 513, 0]), dev([1, 1]), 2, 128, table, 2 ** 24 + 8, dev([7, 8]), 2, dev([0]), *out[:4], 4, out[4])
    w4a8.device_status()
    assert out[0].tolist() == [2 ** 31 - 512, 1] and out[2].tolist() == [5 * 128 + 127, 7 * 128, -1, -1] and out[4].tolist() == [1, 0, 1, 2]
