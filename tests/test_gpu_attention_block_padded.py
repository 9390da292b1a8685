"""A padded step of the attention block: rows behind the last request's come out as zeros, whatever the buffers held before."""
import importlib

import pytest
import torch

from conftest import to_dev

pytestmark = pytest.mark.gpu


def test_rows_that_no_request_owns(w4a8, oracle, cuda):
    mod = importlib.import_module(w4a8.__name__ + ".attention_block")
    hidden, Hq, Hkv, D, R = 256, 4, 2, 64, 3
    tables = mod.PagedTables(R, 8, 40, 16, cuda)
    wqkv, wo = [tuple(to_dev(a, cuda) for a in oracle.make_weights(N, K, 7 + N)) for N, K in (((Hq + 2 * Hkv) * D, hidden), (hidden, Hq * D))]
    layer = mod.AttentionBlock(wqkv, wo, hidden, Hq, Hkv, D, tables, 64)
    layer.mix.fill_(5.0)
    for new, T in (([3, 0, 2], 9), ([30, 4, 20], 54), ([1, 2, 1], 64)):
        X = torch.from_numpy(oracle.make_activations(T, hidden, T)).to(cuda)
        tables.step(torch.tensor(new, dtype=torch.int32, device=cuda), T)
        Y = layer(X, max_q=max(new))
        tables.done()
        w4a8.device_status()
        assert (Y[: sum(new)].abs().amax(dim=1) > 0).all()
        assert (Y[sum(new):] == 0).all()
