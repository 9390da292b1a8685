"""The attention block (plan, QKV product, append, attention, output product) step by step against the plain forms of its parts.

Codes and scales are equal to the plain ones.  The tolerance of the attended rows is that of the attention tests: scores within
reach * 2^-23 * (dim / 16 + 8), weights within that and 2^-18, sums over the keys within 2^-18.
"""
import importlib

import numpy as np
import pytest
import torch

import kv_plain
from conftest import to_dev

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window,softcap", [(0, 0.0), (24, 30.0)])
def test_steps(w4a8, oracle, cuda, window, softcap):
    """Prompts, a request without rows, single tokens, one that the tables have no room for and that comes again with less."""
    mod = importlib.import_module(w4a8.__name__ + ".attention_block")
    hidden, Hq, Hkv, D, block, width, R = 256, 6, 2, 64, 16, 8, 5
    tables = mod.PagedTables(R, width, 40, block, cuda)
    weights = [oracle.make_weights(N, K, 3 + N) for N, K in (((Hq + 2 * Hkv) * D, hidden), (hidden, Hq * D))]
    wqkv, wo = [tuple(to_dev(a, cuda) for a in w) for w in weights]
    layer = mod.AttentionBlock(wqkv, wo, hidden, Hq, Hkv, D, tables, 256, window=window, softcap=softcap)
    codes = [np.zeros((40, Hkv, block, D), np.int8) for _ in range(2)]
    scales = [np.zeros((40, Hkv), np.float32) for _ in range(2)]
    table, kv_len, first, free = np.full((R, width), -1, np.int32), np.zeros(R, np.int32), 0, np.arange(40, dtype=np.int32)
    for step, new in enumerate(([40, 1, 0, 130, 7], [1, 1, 3, 20, 1], [1, 1, 1, 1, 1], [0, 30, 1, 0, 70])):
        T = sum(new)
        X = torch.from_numpy(oracle.make_activations(T, hidden, 50 + step)).to(cuda)
        tables.step(torch.tensor(new, dtype=torch.int32, device=cuda), T)
        Y = layer(X, max_q=max(new))
        tables.done()
        w4a8.device_status()
        want = kv_plain.plan(kv_len, new, block, table, free, first, T)
        assert np.array_equal(tables.slot.cpu().numpy(), want["slot"]) and np.array_equal(tables.table.cpu().numpy(), want["table"])
        table, first, cu, seq = want["table"], int(want["status"][0]), want["cu"], want["seq_len"]
        kv_len = np.where(seq > 0, seq, kv_len).astype(np.int32)
        assert np.array_equal(tables.kv_len.cpu().numpy(), kv_len)
        rows = layer.qkv[:T].cpu().numpy().reshape(T, Hq + 2 * Hkv, D)
        for side in range(2):
            kv_plain.append(rows[:, Hq + side * Hkv:][:, :Hkv], want["slot"], codes[side], scales[side])
        for t, a in zip(layer.cache._tensors, codes + scales):
            assert np.array_equal(t.cpu().numpy(), a)
        k, v = ([kv_plain.rows_of(c, s, table[r], int(n)) for r, n in enumerate(seq)] for c, s in zip(codes, scales))
        o, _, reach = kv_plain.attention(rows[:, :Hq].astype(np.float64), cu, seq, k, v, D ** -0.5, window=window, softcap=softcap)
        vmax = max(float(np.abs(x).max()) for x in v if x.size)
        weight = reach * 2.0 ** -23 * (D / 16 + 8) + 2.0 ** -18
        got = layer.mix[:T].cpu().numpy().reshape(T, Hq, D)
        assert (np.abs(got - o) <= 2 * (weight + 2.0 ** -18) * vmax + 2.0 ** -23 * np.abs(o)).all()
        again = torch.empty_like(Y)
        w4a8.linear(layer.mix, layer.xq, layer.xs, layer.xsum, *wo, again, T, hidden, Hq * D)
        assert torch.equal(again, Y)
