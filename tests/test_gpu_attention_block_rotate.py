"""The attention block with a caller's rotation between the QKV product and the append: what is stored and attended is what it left, and
the positions that it gets are the rows' places in their requests."""
import importlib

import numpy as np
import pytest
import torch

import kv_plain
from conftest import to_dev

pytestmark = pytest.mark.gpu


def rotary(x, position):
    """Pairs (i, i + dim / 2) by position * 10000^(-2i / dim), in place."""
    half = x.shape[2] // 2
    a = position.clamp(min=0)[:, None].double() * 10000.0 ** (-torch.arange(half, device=x.device, dtype=torch.float64) / half)
    c, s = a.cos()[:, None].float(), a.sin()[:, None].float()
    u, v = x[..., :half].clone(), x[..., half:].clone()
    x[..., :half] = u * c - v * s
    x[..., half:] = u * s + v * c


def test_rotated_rows_are_stored(w4a8, oracle, cuda):
    mod = importlib.import_module(w4a8.__name__ + ".attention_block")
    hidden, Hq, Hkv, D, block, R = 256, 4, 2, 64, 16, 3
    seen = []

    def rotate(q, k, position):
        seen.append((q.shape, k.shape, position.clone(), q.clone(), k.clone()))
        rotary(q, position)
        rotary(k, position)
    tables = mod.PagedTables(R, 6, 30, block, cuda)
    wqkv, wo = [tuple(to_dev(a, cuda) for a in oracle.make_weights(N, K, 5 + N)) for N, K in (((Hq + 2 * Hkv) * D, hidden), (hidden, Hq * D))]
    layer = mod.AttentionBlock(wqkv, wo, hidden, Hq, Hkv, D, tables, 64, rotate=rotate)
    codes, scales = [np.zeros((30, Hkv, block, D), np.int8) for _ in range(2)], [np.zeros((30, Hkv), np.float32) for _ in range(2)]
    kv_len, table, first = np.zeros(R, np.int32), np.full((R, 6), -1, np.int32), 0
    for new in ([20, 1, 9], [1, 1, 3]):
        T = sum(new)
        X = torch.from_numpy(oracle.make_activations(T, hidden, T)).to(cuda)
        tables.step(torch.tensor(new, dtype=torch.int32, device=cuda), T)
        layer(X, max_q=max(new))
        tables.done()
        w4a8.device_status()
        want = kv_plain.plan(kv_len, new, block, table, np.arange(30, dtype=np.int32), first, T)
        table, first, kv_len = want["table"], int(want["status"][0]), want["seq_len"]
        q_shape, k_shape, position, q, k = seen[-1]
        assert q_shape == (T, Hq, D) and k_shape == (T, Hkv, D) and np.array_equal(position.cpu().numpy(), want["position"])
        rotary(q, position)
        rotary(k, position)
        rows = layer.qkv[:T].view(T, Hq + 2 * Hkv, D)
        assert torch.equal(rows[:, :Hq], q) and torch.equal(rows[:, Hq:Hq + Hkv], k)
        host = rows.cpu().numpy()
        for side in range(2):
            kv_plain.append(host[:, Hq + side * Hkv:][:, :Hkv], want["slot"], codes[side], scales[side])
        for t, a in zip(layer.cache._tensors, codes + scales):
            assert np.array_equal(t.cpu().numpy(), a)
    assert len(seen) == 2
