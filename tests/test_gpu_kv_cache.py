"""GPU tests of the 8-bit KV cache's plan, write and read against the plain forms: integers and codes equal, scales bit for bit."""
import numpy as np
import pytest
import torch

import kv_plain
from conftest import to_dev

pytestmark = pytest.mark.gpu
DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def plan_on_gpu(w, cuda, kv, new, block, table, free, first, rows, position=True):
    kv_d, new_d = to_dev(np.asarray(kv, np.int32), cuda), to_dev(np.asarray(new, np.int32), cuda)
    R = len(kv)
    out = {"table": to_dev(table, cuda), "seq_len": torch.full((R,), -9, dtype=torch.int32, device=cuda), "cu": torch.full((R + 1,), -9, dtype=torch.int32, device=cuda),
           "slot": torch.full((rows + 5,), -9, dtype=torch.int32, device=cuda), "position": torch.full((rows + 5,), -9, dtype=torch.int32, device=cuda),
           "status": torch.zeros(4, dtype=torch.int32, device=cuda)}
    free_d = to_dev(np.asarray(free if len(free) else [0], np.int32), cuda)
    w.kv_plan(kv_d, new_d, R, block, out["table"], table.shape[1], free_d, len(free), to_dev(np.array([first], np.int32), cuda), out["seq_len"], out["cu"],
              out["slot"], out["position"] if position else None, rows, out["status"])
    w.device_status()
    got = {k: v.cpu().numpy() for k, v in out.items()}
    assert (got["slot"][rows:] == -9).all() and (got["position"][rows:] == -9).all()       # nothing written behind the rows
    got["slot"], got["position"] = got["slot"][:rows], got["position"][:rows]
    return got


def tables(rng, kv, block, width, extra):
    need = [-(-max(0, int(k)) // block) for k in kv]
    ids = rng.permutation(sum(min(n, width) for n in need) + extra).astype(np.int32)
    table, at = np.full((len(kv), width), -1, np.int32), 0
    for r, n in enumerate(need):
        n = min(n, width)
        table[r, :n] = ids[at:at + n]
        at += n
    return table, ids[at:]


@pytest.mark.parametrize("R,block,lo,hi,new_hi,first,short,pad", [
    (1, 16, 0, 0, 1, 0, 0, 0), (1, 16, 15, 15, 1, 0, 0, 3), (1, 16, 16, 16, 1, 0, 0, 0), (1, 64, 0, 0, 700, 0, 0, 1), (3, 16, 0, 40, 2, 1, 1, 2),
    (33, 32, 0, 500, 1, 4, 0, 0), (257, 16, 0, 100, 5, 0, 1, 7), (511, 128, 0, 3000, 300, 2, 0, 0), (512, 16, 5, 60, 1, 0, 1, 9), (513, 16, 0, 60, 3, 0, 0, -20),
    (4097, 64, 0, 900, 40, 3, 1, 11), (16384, 16, 0, 33, 2, 0, 1, 0),
])
def test_plan(w4a8, cuda, R, block, lo, hi, new_hi, first, short, pad):
    rng = np.random.default_rng(R * 1000 + block)
    kv, new = rng.integers(lo, hi + 1, R).astype(np.int32), rng.integers(0 if R > 1 else new_hi, new_hi + 1, R).astype(np.int32)
    need = int(((kv + new + block - 1) // block - (kv + block - 1) // block).sum())
    width = int((-(-(kv + new) // block)).max()) + 1
    table, spare = tables(rng, kv, block, width, need + 8)
    free = spare[: first + (need * 2 // 3 if short else need + 3)]
    rows = max(0, int(new.sum()) + pad)                                       # negative pad: the step's rows do not hold all tokens
    want = kv_plain.plan(kv, new, block, table, free, first, rows)
    got = plan_on_gpu(w4a8, cuda, kv, new, block, table, free, first, rows)
    for k in want:
        assert np.array_equal(got[k], want[k]), k


def test_plan_odd_inputs(w4a8, cuda):
    """Negative lengths count as none; a request longer than its table row is not served and takes no block from those behind it; an empty
    free list still serves requests that need nothing; no request at all."""
    table = np.array([[3, -1], [5, 6], [-1, -1], [7, -1]], np.int32)
    kv, new = [-4, 30, 0, 10], [2, 3, -1, 6]
    free = [11, 12]
    want = kv_plain.plan(kv, new, 16, table, free, 0, 12)
    assert want["status"].tolist() == [1, 1, 1, 8]
    got = plan_on_gpu(w4a8, cuda, kv, new, 16, table, free, 0, 12)
    for k in want:
        assert np.array_equal(got[k], want[k]), k
    got = plan_on_gpu(w4a8, cuda, [3, 16], [1, 1], 16, np.array([[2, -1], [4, -1]], np.int32), [], 0, 2, position=False)
    assert got["seq_len"].tolist() == [4, 0] and got["slot"].tolist() == [35, -1] and got["status"].tolist() == [0, 1, 0, 1]
    got = plan_on_gpu(w4a8, cuda, [], [], 16, np.zeros((0, 1), np.int32), [1], 0, 4)
    assert got["cu"].tolist() == [0] and got["slot"].tolist() == [-1] * 4 and got["status"].tolist() == [0, 0, 0, 0]


def pool(rng, blocks, heads, block, dim):
    return [rng.integers(-127, 128, (blocks, heads, block, dim)).astype(np.int8) for _ in range(2)] + \
           [(rng.random((blocks, heads)) * 0.02 + 0.005).astype(np.float32) for _ in range(2)]


def write_on_gpu(w, cuda, k, v, slot, arrays, dtype, pad=0, stream=None):
    """The rows as columns of a wider tensor; returns the cache's four arrays after the call."""
    T, heads, dim = k.shape
    wide = torch.full((T, 2 * heads * dim + pad), 7.0, dtype=DT[dtype], device=cuda)
    wide[:, : heads * dim] = to_dev(k.reshape(T, -1), cuda).to(DT[dtype])
    wide[:, heads * dim: 2 * heads * dim] = to_dev(v.reshape(T, -1), cuda).to(DT[dtype])
    dev = [to_dev(a, cuda) for a in arrays]
    cache = w.KVCache.of(*dev)
    torch.cuda.synchronize()
    w.launch_kv_append_q8(wide, wide[:, heads * dim:], wide.shape[1], to_dev(np.asarray(slot, np.int32), cuda), T, cache, dtype, stream=stream)
    w.device_status()
    return [d.cpu().numpy() for d in dev], cache, wide


def rounded(x, dtype):
    return torch.from_numpy(x).to(DT[dtype]).float().numpy()


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("heads,block,dim,runs", [
    (1, 16, 64, [(0, 0, 1)]), (2, 16, 128, [(1, 15, 1), (0, 0, 16), (4, 7, 9)]), (3, 32, 64, [(2, 31, 1), (5, 1, 30), (0, 0, 5), (1, 0, 32)]),
    (8, 16, 128, [(i, (i * 7) % 16, 1) for i in range(40)]), (2, 64, 256, [(0, 3, 61), (1, 0, 64), (2, 63, 1)]), (1, 128, 256, [(3, 0, 128), (1, 127, 1), (0, 5, 100)]),
    (5, 16, 64, [(i, 0, 16) for i in range(33)]), (1, 128, 64, [(2, 64, 64), (0, 0, 128)]),
])
def test_append(w4a8, cuda, dtype, heads, block, dim, runs):
    rng = np.random.default_rng(heads * 100 + block + dim)
    blocks = max(b for b, _, _ in runs) + 2
    arrays = pool(rng, blocks, heads, block, dim)
    slot = np.concatenate([b * block + np.arange(o, o + m) for b, o, m in runs] + [np.array([-1, -1])])
    slot = np.insert(slot, 1, -1) if runs[0][2] == 1 else slot                       # a padded row between two runs
    k, v = (rng.standard_normal((len(slot), heads, dim)).astype(np.float32) * rng.choice([0.3, 1.0, 3.0], (len(slot), heads, 1)).astype(np.float32) for _ in range(2))
    got, cache, _ = write_on_gpu(w4a8, cuda, k, v, slot, arrays, dtype, pad=8)
    want = [a.copy() for a in arrays]
    kv_plain.append(rounded(k, dtype), slot, want[0], want[2])
    kv_plain.append(rounded(v, dtype), slot, want[1], want[3])
    assert np.array_equal(got[2], want[2]) and np.array_equal(got[3], want[3])
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def test_append_values_that_are_not_ordinary(w4a8, cuda):
    """Zeros (scale 0, then a later token gives the block its scale), an infinity (its block's scale is infinite, other heads and blocks are not
    touched), NaN (stored as 0, no part in the scale), subnormal and huge numbers."""
    rng = np.random.default_rng(5)
    arrays = pool(rng, 6, 2, 16, 64)
    k = rng.standard_normal((8, 2, 64)).astype(np.float32)
    k[0] = 0.0
    k[2, 0, 5] = np.inf
    k[3, 1, 7] = np.nan
    k[4] *= 1e-40
    k[5] *= 1e37
    slot = np.array([0, 1, 16 + 3, 32, 48, 64, -1, 80])
    got, cache, wide = write_on_gpu(w4a8, cuda, k, k, slot, arrays, "fp32")
    want = [a.copy() for a in arrays]
    kv_plain.append(k, slot, want[0], want[2])
    kv_plain.append(k, slot, want[1], want[3])
    assert np.isinf(want[2][1, 0]) and np.isfinite(want[2][1, 1]) and np.isfinite(want[2][2]).all()
    for a, b in zip(got, want):
        assert np.array_equal(a, b)


def test_append_a_token_at_a_time_and_again(w4a8, cuda):
    """A block filled token by token with growing numbers: each step rounds the codes in front to the new scale, as the plain form does; a call
    that is made twice changes nothing the second time."""
    rng = np.random.default_rng(6)
    arrays = pool(rng, 2, 2, 16, 128)
    want = [a.copy() for a in arrays]
    for t in range(16):
        k = (rng.standard_normal((1, 2, 128)) * 1.3 ** t).astype(np.float32)
        for again in range(2):
            arrays, _, _ = write_on_gpu(w4a8, cuda, k, -k, [16 + t], arrays, "fp32")
            kv_plain.append(k, [16 + t], want[0], want[2])
            kv_plain.append(-k, [16 + t], want[1], want[3])
            for a, b in zip(arrays, want):
                assert np.array_equal(a, b), t


def test_append_slot_beyond_the_cache_is_reported(w4a8, cuda):
    rng = np.random.default_rng(7)
    arrays = pool(rng, 2, 1, 16, 64)
    k = rng.standard_normal((3, 1, 64)).astype(np.float32)
    with pytest.raises(w4a8.W4A8Error) as e:
        write_on_gpu(w4a8, cuda, k, k, [3, 32, 2 ** 31 - 1], arrays, "fp32")
    assert e.value.code == w4a8.ERR_DEVICE and "slot" in str(e.value)
    w4a8.device_status()                                                              # reported once


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("heads,block,dim,lens", [(1, 16, 64, [1]), (2, 16, 128, [17, 0, 64, 5]), (8, 64, 256, [65, 200]), (4, 128, 128, [3] * 70), (3, 32, 64, [1000])])
def test_read(w4a8, cuda, dtype, heads, block, dim, lens):
    rng = np.random.default_rng(block + dim + len(lens))
    begin = np.array([(7 * i) % 50 for i in range(len(lens))], np.int32)
    ends = begin + np.array(lens)
    width = int((-(-ends // block)).max()) + 1
    table, _ = tables(rng, ends, block, width, 3)
    blocks = int(table.max()) + 4
    arrays = pool(rng, blocks, heads, block, dim)
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    T = int(cu[-1])
    pitch = heads * dim + 8
    dev = [to_dev(a, cuda) for a in arrays]
    outs = [torch.full((T + 2, pitch), 5.0, dtype=DT[dtype], device=cuda) for _ in range(2)]
    w4a8.launch_kv_read_q8(w4a8.KVCache.of(*dev), to_dev(table, cuda), width, to_dev(begin, cuda), to_dev(cu, cuda), len(lens), T + 2, outs[0], outs[1], pitch, dtype)
    w4a8.device_status()
    for out, codes, scale in zip(outs, arrays[:2], arrays[2:]):
        assert (out[T:] == 5.0).all() and (out[:, heads * dim:] == 5.0).all()         # rows behind the last, columns beside
        for r, n in enumerate(lens):
            want = kv_plain.rows_of(codes, scale, table[r], int(ends[r]))[begin[r]:]
            got = out[cu[r]:cu[r + 1], : heads * dim].cpu()
            assert torch.equal(got, torch.from_numpy(want.reshape(n, heads * dim)).float().to(DT[dtype]))   # a product of 31 bits at most: fp64 to fp32 rounds it once


def test_read_of_a_block_that_is_not_there_is_reported(w4a8, cuda):
    rng = np.random.default_rng(8)
    dev = [to_dev(a, cuda) for a in pool(rng, 3, 1, 16, 64)]
    out = torch.full((20, 64), 5.0, device=cuda)
    table = to_dev(np.array([[1, 99]], np.int32), cuda)
    w4a8.launch_kv_read_q8(w4a8.KVCache.of(*dev), table, 2, to_dev(np.zeros(1, np.int32), cuda), to_dev(np.array([0, 20], np.int32), cuda), 1, 20, out, out.clone(), 64)
    with pytest.raises(w4a8.W4A8Error) as e:
        w4a8.device_status()
    assert e.value.code == w4a8.ERR_DEVICE and "block table" in str(e.value)
    assert (out[:16] != 5.0).any() and (out[16:] == 5.0).all()


def test_blocks_past_two_to_the_31_bytes(w4a8, cuda):
    """Offsets in a large pool: 1.2 million blocks of 2 KB a side, the last ones in use."""
    rng = np.random.default_rng(9)
    blocks, block, dim = 1_200_000, 16, 128
    k, v = (torch.zeros((blocks, 1, block, dim), dtype=torch.int8, device=cuda) for _ in range(2))
    ks, vs = (torch.zeros((blocks, 1), device=cuda) for _ in range(2))
    cache = w4a8.KVCache.of(k, v, ks, vs)
    x = rng.standard_normal((20, 1, dim)).astype(np.float32)
    b = blocks - 2
    slot = to_dev((b * block + np.arange(20)).astype(np.int32), cuda)
    w4a8.launch_kv_append_q8(to_dev(x, cuda), to_dev(-x, cuda), dim, slot, 20, cache)
    out = [torch.zeros((20, dim), device=cuda) for _ in range(2)]
    table = to_dev(np.array([[b, b + 1]], np.int32), cuda)
    w4a8.launch_kv_read_q8(cache, table, 2, to_dev(np.zeros(1, np.int32), cuda), to_dev(np.array([0, 20], np.int32), cuda), 1, 20, out[0], out[1], dim)
    w4a8.device_status()
    codes, scale = np.zeros((2, 1, block, dim), np.int8), np.zeros((2, 1), np.float32)
    kv_plain.append(x, np.arange(20), codes, scale)
    want = kv_plain.rows_of(codes, scale, [0, 1], 20).reshape(20, dim).astype(np.float32)
    assert np.array_equal(out[0].cpu().numpy(), want) and np.array_equal(out[1].cpu().numpy(), -want)
    assert int(k[:b].abs().amax()) == 0                                               # nothing anywhere else
