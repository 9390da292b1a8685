"""The layer operators together, as a decoder layer runs them (decoder_layer.py), and the attention block with a Rope and 8-bit projections."""
import importlib

import numpy as np
import pytest
import torch

import kv_plain
from conftest import to_dev
from layer_plain import U, add_norm32, near, norm, quantize
from test_gpu_moe_route import plain as plain_route

pytestmark = pytest.mark.gpu
HIDDEN, HQ, HKV, D, BLOCK, R, E, TOPK, INNER = 256, 4, 2, 64, 16, 3, 16, 4, 64


def eight_bit(n, k, seed, dev):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randint(-127, 128, (n, k), generator=g, device=dev, dtype=torch.int8), torch.rand(n, generator=g, device=dev) * 2e-3 + 1e-4)


def product(x, matrix):
    q, scale, _ = quantize(x, 0)
    return (q.double() @ matrix[0].double().T).float() * scale * matrix[1]


def turned(x, position, weight):
    """Norm and rotation of pairs (i, i + D / 2) in 64 bits, and |a| + |b| of each pair."""
    T, H, _ = x.shape
    x = norm(x.double().reshape(T * H, D), weight, 0, 1e-6).view(T, H, D)
    f = 10000.0 ** (-torch.arange(D // 2, device=x.device, dtype=torch.float64) / (D // 2))
    a = position.clamp(min=0)[:, None, None].double() * f
    u, v = x[..., : D // 2], x[..., D // 2:]
    return torch.cat((u * a.cos() - v * a.sin(), v * a.cos() + u * a.sin()), 2), torch.cat((u.abs() + v.abs(),) * 2, 2)


def attention(w4a8, oracle, dev, q_w, k_w):
    mod = importlib.import_module(w4a8.__name__ + ".attention_block")
    tables = mod.PagedTables(R, 6, 30, BLOCK, dev)
    rope = w4a8.Rope.of(D, D, 10000.0, q_weight=q_w, k_weight=k_w, variant=0, device=dev)
    wqkv = tuple(to_dev(a, dev) for a in oracle.make_weights((HQ + 2 * HKV) * D, HIDDEN, 5))
    return tables, mod.AttentionBlock(wqkv, eight_bit(HIDDEN, HQ * D, 6, dev), HIDDEN, HQ, HKV, D, tables, 64, rotate=rope)


STEPS = ([20, 1, 9], [1, 1, 3], [1, 0, 1])


def weights_of_norms(dev):
    g = torch.Generator(device=dev).manual_seed(1)
    return [torch.randn(n, generator=g, device=dev) * 0.1 + 1 for n in (D, D, HIDDEN, HIDDEN)]


def test_attention_block_with_a_rope_and_eight_bit_weights(w4a8, oracle, cuda):
    q_w, k_w, _, _ = weights_of_norms(cuda)
    tables, block = attention(w4a8, oracle, cuda, q_w, k_w)
    codes, scales = [np.zeros((30, HKV, BLOCK, D), np.int8) for _ in range(2)], [np.zeros((30, HKV), np.float32) for _ in range(2)]
    for new in STEPS:
        T = sum(new) + 2                                              # two rows that no request owns
        X = torch.from_numpy(oracle.make_activations(T, HIDDEN, T)).to(cuda)
        slot = tables.step(torch.tensor(new, dtype=torch.int32, device=cuda), T)
        Y = block(X, max_q=max(new))
        w4a8.device_status()
        raw = torch.empty_like(block.qkv)
        w4a8.linear(X, torch.empty_like(block.xq), torch.empty_like(block.xs), torch.empty_like(block.xsum), *block.wqkv, raw, T, block.cols, HIDDEN)
        rows, raw = block.qkv[:T].view(T, -1, D), raw[:T].view(T, -1, D)
        there = tables.position >= 0
        assert torch.equal(rows[~there], raw[~there]) and torch.equal(rows[:, HQ + HKV:], raw[:, HQ + HKV:])
        for lo, n, w in ((0, HQ, q_w), (HQ, HKV, k_w)):
            want, size = turned(raw[:, lo:lo + n], tables.position, w)
            near(rows[:, lo:lo + n][there], want[there], 20 * U * size[there], "turned")
        host = rows.cpu().numpy()
        for side in range(2):
            kv_plain.append(host[:, HQ + side * HKV:][:, :HKV], slot.cpu().numpy(), codes[side], scales[side])
        for t, a in zip(block.cache._tensors, codes + scales):
            assert np.array_equal(t.cpu().numpy(), a)
        assert torch.equal(Y, product(block.mix[:T], block.wo)) and (Y[~there] == 0).all()
        tables.done()


def layer_of(w4a8, oracle, dev, norms):
    mod = importlib.import_module(w4a8.__name__ + ".decoder_layer")
    tables, block = attention(w4a8, oracle, dev, norms[0], norms[1])
    gate_up, down = [tuple(to_dev(a, dev) for a in oracle.make_weights(E * n, k, 9 + n)) for n, k in ((2 * INNER, HIDDEN), (HIDDEN, INNER))]
    return tables, mod.DecoderLayer(block, w4a8.Norm.of(HIDDEN, norms[2], 0), w4a8.Norm.of(HIDDEN, norms[3], 0, alpha=0.5), w4a8.Router.of(E, TOPK, groups=4, topk_groups=2, group_score="sum2"),
                                    eight_bit(E, HIDDEN, 12, dev), gate_up, down, INNER)


def test_the_operators_of_a_layer_one_after_the_other(w4a8, oracle, cuda):
    norms = weights_of_norms(cuda)
    tables, layer = layer_of(w4a8, oracle, cuda, norms)
    other_tables, other = attention(w4a8, oracle, cuda, norms[0], norms[1])
    for new in STEPS:
        T = sum(new) + 2
        g = torch.Generator(device="cuda").manual_seed(T)
        h = torch.randn(T, HIDDEN, generator=g, device=cuda)
        y = None if new is STEPS[0] else torch.randn(T, HIDDEN, generator=g, device=cuda)
        h_start = h.clone()
        lengths = torch.tensor(new, dtype=torch.int32, device=cuda)
        tables.step(lengths, T)
        out = layer(h, y, max_q=max(new))
        # the same with plain forms of the new operators, and the attention and expert blocks by themselves
        other_tables.step(lengths, T)
        s, n = add_norm32(h_start, y, norms[2], 0, None, -1, None, 1.0, 1e-6)
        a = other(n, max_q=max(new))
        s, n = add_norm32(s, a, norms[3], 0, None, -1, None, 0.5, 1e-6)
        assert torch.equal(h, s) and torch.equal(layer.normed[:T], n)
        logits = product(n, layer.router_w)
        assert torch.equal(layer.logits[:T], logits)
        idx, weight = plain_route(logits, TOPK, groups=4, topk_groups=2, group_score="sum2")
        assert np.array_equal(layer.idx[:T].cpu().numpy(), idx) and np.allclose(layer.weight[:T].cpu().numpy(), weight, rtol=22 * U, atol=U)
        want = torch.empty_like(out)
        w4a8.moe_block(n, *layer.gate_up, *layer.down, layer.idx, layer.weight, want, T, TOPK, HIDDEN, INNER, E, torch.empty_like(layer.workspace))
        assert torch.equal(out, want) and torch.isfinite(out).all()
        w4a8.device_status()
        tables.done()
        other_tables.done()


def test_a_layer_in_a_graph(w4a8, oracle, cuda):
    """A decode step captured and replayed with new rows gives what the calls give."""
    norms, T = weights_of_norms(cuda), 3
    (tables, layer), (plain_tables, plain) = (layer_of(w4a8, oracle, cuda, norms) for _ in range(2))
    h, y = torch.randn(T, HIDDEN, device=cuda), torch.randn(T, HIDDEN, device=cuda)
    ones = torch.ones(R, dtype=torch.int32, device=cuda)
    tables.step(ones, T)
    plain_tables.step(ones, T)
    plain(h.clone(), y, max_q=1)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        layer(h.clone(), y, max_q=1)                                  # a call of each kernel before the capture
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(h, y, max_q=1)
    for seed in range(3):
        g = torch.Generator(device="cuda").manual_seed(seed)
        h.copy_(torch.randn(T, HIDDEN, generator=g, device=cuda))
        y.copy_(torch.randn(T, HIDDEN, generator=g, device=cuda))
        h2 = h.clone()
        graph.replay()
        want = plain(h2, y, max_q=1)
        assert torch.equal(out, want) and torch.equal(h, h2)
    w4a8.device_status()


def test_a_step_without_rows(w4a8, oracle, cuda):
    tables, layer = layer_of(w4a8, oracle, cuda, weights_of_norms(cuda))
    tables.step(torch.zeros(R, dtype=torch.int32, device=cuda), 0)
    empty = torch.empty(0, HIDDEN, device=cuda)
    assert layer(empty).shape == (0, HIDDEN) and layer(empty, empty.clone()).shape == (0, HIDDEN)
    tables.done()
    assert (tables.kv_len == 0).all() and w4a8.device_status() is None
