"""GPU tests of attention over the 8-bit KV cache against the plain form in 64 bits.

Tolerance, from the number formats alone.  A score is a sum of dim products, each exact to 2^-22 (fp32 rows: two fp16 terms) or exact (16-bit
rows), added in fp32 in at most dim / 16 + 2 roundings of 2^-23 of what is summed so far, then scaled twice: its error is at most
A * 2^-23 * (dim / 16 + 8) with A = scale * sum |q| |k|.  A weight's relative error is that plus 2^-21 (exp2, its argument's rounding at
magnitudes up to 64: 2^-18), and 2^-11 for the fp16 rounding of 16-bit rows.  The numerator and the denominator each carry it once, the
fp32 sums over the keys add 2^-18: |o - o'| <= 2 * weight error * max |v|.  (Requests of few rows: an element is held to 2^-24 of its row's largest
magnitude and everything behind it is exact, which stays within A * 2^-23 * (dim / 16 + 8) while that largest is at most 2 * (dim / 16 + 8) = 24 times
the rows' mean magnitude weighted by the keys; normally distributed rows have 4.)  16-bit results add their own rounding, 2^-11 or 2^-8 of |o|.
"""
import numpy as np
import pytest
import torch

import kv_plain
from conftest import to_dev

pytestmark = pytest.mark.gpu
DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


class Case:
    """Requests with `seqs` tokens, the last news[r] of them queries, over a pool in random order: blocks that no request holds have scales that
    are not numbers, table entries behind a request's blocks name none, Q and O are columns of wider tensors."""

    def __init__(self, w, cuda, seqs, news, Hq, Hkv, D, block, dtype="fp32", causal=1, window=0, softcap=0.0, seed=1, sharp=1.5, pad_rows=2, magnitude=0.7):
        rng = np.random.default_rng(seed)
        self.w, self.cuda, self.seqs, self.news, self.Hq, self.D, self.dtype = w, cuda, np.array(seqs, np.int32), np.array(news), Hq, D, dtype
        self.kw = dict(causal=causal, window=window, softcap=softcap)
        self.cu = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        self.T = int(self.cu[-1]) + pad_rows
        need = [-(-s // block) for s in seqs]
        self.width = max(1, max(need)) + 1
        ids = rng.permutation(sum(need) + 3).astype(np.int32)
        self.table, at = np.full((len(seqs), self.width), -1, np.int32), 0
        for r, n in enumerate(need):
            self.table[r, :n] = ids[at:at + n]
            at += n
        blocks = len(ids)
        self.k, self.v = (np.clip(np.rint(rng.standard_normal((blocks, Hkv, block, D)) * 38), -127, 127).astype(np.int8) for _ in range(2))
        self.ks, self.vs = ((np.exp(magnitude * rng.standard_normal((blocks, Hkv))) / 45).astype(np.float32) for _ in range(2))
        for s in (self.ks, self.vs):
            s[ids[at:]] = np.nan
        q = rng.standard_normal((self.T, Hq, D)).astype(np.float32) * sharp
        self.q = torch.from_numpy(q).to(DT[dtype])
        self.scale = D ** -0.5

    def run(self, max_q=None, stream=None, lse=True, workspace=None):
        w, cuda, Hq, D = self.w, self.cuda, self.Hq, self.D
        cols = Hq * D
        wide = torch.full((self.T, cols + 24), 3.0, dtype=DT[self.dtype], device=cuda)
        wide[:, 8:8 + cols] = self.q.reshape(self.T, cols).to(cuda)
        out = torch.full((self.T, cols + 16), 3.0, dtype=DT[self.dtype], device=cuda)
        ls = torch.full((self.T, Hq), 3.0, device=cuda) if lse else None
        dev = [to_dev(a, cuda) for a in (self.k, self.v, self.ks, self.vs)]
        cache = w.KVCache.of(*dev)
        table, cu, seqs = (to_dev(a, cuda) for a in (self.table, self.cu, self.seqs))
        mq = max(int(n) for n in self.news) if max_q is None else max_q
        if workspace is None:
            workspace = torch.zeros(w.attention_q8_workspace_bytes(Hq, cache, self.T, mq), dtype=torch.uint8, device=cuda)
        torch.cuda.synchronize()
        w.launch_attention_q8(wide[:, 8:], cols + 24, cache, table, self.width, cu, seqs, len(self.seqs), self.T, Hq, out, cols + 16, self.scale, self.dtype,
                              workspace, max_q=mq, lse=ls, stream=stream, **self.kw)
        w.device_status()
        assert (out[:, cols:] == 3.0).all() and (out[self.cu[-1]:] == 3.0).all()       # columns beside, rows behind
        if lse:
            assert (ls[self.cu[-1]:] == 3.0).all()
        return out[: self.cu[-1], :cols].reshape(-1, Hq, D).float().cpu().numpy(), ls[: self.cu[-1]].cpu().numpy() if lse else None

    def plain(self):
        k, v = ([kv_plain.rows_of(c, s, self.table[r], int(n)) for r, n in enumerate(self.seqs)] for c, s in ((self.k, self.ks), (self.v, self.vs)))
        vmax = max([float(np.abs(x[np.isfinite(x)]).max()) for x in v if x.size] or [0.0])
        o, l, reach = kv_plain.attention(self.q[: self.cu[-1]].double().numpy(), self.cu, self.seqs, k, v, self.scale, **self.kw)
        return o, l, reach, vmax

    def tolerance(self, reach, vmax, o):
        score = reach * 2.0 ** -23 * (self.D / 16 + 8)
        weight = score + 2.0 ** -18 + (0 if self.dtype == "fp32" else 2.0 ** -11)
        out = {"fp32": 2.0 ** -23, "fp16": 2.0 ** -11, "bf16": 2.0 ** -8}[self.dtype]
        return 2 * (weight + 2.0 ** -18) * vmax + out * np.abs(o), score + 2.0 ** -16

    def check(self, **kw):
        got, lse = self.run(**kw)
        o, l, reach, vmax = self.plain()
        tol, tol_l = self.tolerance(reach, vmax, o)
        assert np.isfinite(got).all()
        assert (np.abs(got - o) <= tol).all(), float((np.abs(got - o) - tol).max())
        if lse is not None:
            assert np.array_equal(np.isneginf(lse), np.isneginf(l))
            there = np.isfinite(l)
            assert (np.abs(lse[there] - l[there]) <= tol_l * (1 + np.abs(l[there]))).all()
        return got


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_decode(w4a8, cuda, dtype, D, block):
    """Lengths around tiles and blocks, one new token each."""
    Case(w4a8, cuda, [1, 2, 15, 16, 17, 63, 64, 65, 127, 129, 200, 513], [1] * 12, 8, 2, D, block, dtype, seed=D + block).check()


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (2, 2), (3, 1), (7, 1), (8, 1), (9, 1), (14, 2), (16, 1), (17, 1), (33, 1), (64, 2)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_decode_head_groups(w4a8, cuda, Hq, Hkv, dtype):
    Case(w4a8, cuda, [5, 100, 333], [1, 1, 1], Hq, Hkv, 128, 16, dtype, seed=Hq).check()


@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
@pytest.mark.parametrize("D,Hq,Hkv", [(64, 8, 2), (128, 12, 4), (128, 7, 1), (256, 4, 2)])
def test_few_queries(w4a8, cuda, dtype, D, Hq, Hkv):
    """One to eight queries a request, none in one, more queries than that fit a tile of rows."""
    Case(w4a8, cuda, [9, 64, 70, 300, 129, 40], [1, 8, 3, 5, 0, 11], Hq, Hkv, D, 16, dtype, seed=D + Hq).check()


@pytest.mark.parametrize("causal,window,softcap", [(1, 1, 0.0), (1, 16, 0.0), (1, 100, 30.0), (0, 0, 0.0), (0, 50, 0.0), (0, 0, 5.0), (1, 10 ** 9, 0.0)])
@pytest.mark.parametrize("D,news", [(64, [1, 1, 1, 1]), (128, [4, 1, 6, 2]), (256, [1, 2, 1, 1]), (128, [40, 1, 100, 64])])
def test_masks(w4a8, cuda, causal, window, softcap, D, news):
    Case(w4a8, cuda, [40, 66, 400, 131], news, 4, 2, D, 16, "fp32", causal, window, softcap, seed=window % 1000 + D).check()


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("D,Hq,Hkv,block,seqs,news", [
    (128, 4, 1, 16, [64], [64]), (128, 2, 2, 64, [300], [300]), (64, 8, 2, 16, [129, 500], [129, 37]), (256, 4, 2, 32, [200, 70], [200, 33]),
    (128, 8, 2, 128, [33, 1, 257, 600], [33, 1, 200, 65]), (128, 5, 1, 16, [130, 90], [130, 64]),
])
def test_prompts(w4a8, cuda, dtype, D, Hq, Hkv, block, seqs, news):
    Case(w4a8, cuda, seqs, news, Hq, Hkv, D, block, dtype, seed=sum(seqs)).check()


def test_prompts_masked(w4a8, cuda):
    for dtype, causal, window, softcap in (("fp32", 1, 70, 0.0), ("bf16", 0, 0, 0.0), ("fp16", 1, 33, 20.0), ("fp32", 0, 40, 0.0)):
        Case(w4a8, cuda, [300, 140], [200, 140], 4, 2, 128, 16, dtype, causal, window, softcap, seed=window).check()


def test_requests_without_tokens_or_queries(w4a8, cuda):
    """seq_len 0 (a request that the plan did not serve) gives zeros, with any number of rows; more rows than tokens: those in front see nothing."""
    for news in ([1, 1, 2], [3, 1, 100]):
        c = Case(w4a8, cuda, [0, 40, 0], news, 4, 2, 64, 16)
        got = c.check()
        assert (got[: news[0]] == 0).all() and (got[news[0] + 1:] == 0).all()
    Case(w4a8, cuda, [3, 5], [7, 90], 4, 2, 128, 16).check()


@pytest.mark.parametrize("news", [3, 100])
def test_infinite_block_behind_the_mask(w4a8, cuda, news):
    """A block with infinite scales (an infinity was written) is not a number to the queries that see it and nothing to those before it."""
    c = Case(w4a8, cuda, [64 + news], [news], 4, 2, 128, 16, seed=3)
    bad = c.table[0, (64 + news - 1) // 16]
    c.ks[bad] = c.vs[bad] = np.inf
    got, _ = c.run()
    first = (64 + news - 1) // 16 * 16 - 64                    # the first query that sees the block
    assert np.isnan(got[max(first, 0):]).any(axis=(1, 2)).all()
    if first > 0:
        assert np.isfinite(got[:first]).all()
        c.ks[bad] = c.vs[bad] = 1.0
        assert np.array_equal(got[:first], c.run()[0][:first])


def test_queries_that_are_not_numbers_stay_alone(w4a8, cuda):
    c = Case(w4a8, cuda, [100, 90], [2, 80], 4, 2, 128, 16, seed=4)
    o, _, reach, vmax = c.plain()
    c.q[1, 2] = float("nan")
    c.q[20, 0, 5] = float("inf")
    got = c.run()[0]
    assert np.isnan(got[1, 2]).all() and np.isnan(got[20, 0]).any()
    got[1, 2], got[20, 0] = o[1, 2], o[20, 0]
    assert (np.abs(got - o) <= c.tolerance(reach, vmax, o)[0]).all()


@pytest.mark.parametrize("magnitude,sharp", [(3.0, 1.0), (0.0, 30.0), (6.0, 0.1)])
def test_uneven_scales_and_peaked_scores(w4a8, cuda, magnitude, sharp):
    """Blocks whose scales differ by factors of thousands, scores of hundreds: the running maximum and the weights' reference move often."""
    c = Case(w4a8, cuda, [700, 333], [1, 70], 8, 2, 128, 16, seed=11, magnitude=magnitude, sharp=sharp)
    if magnitude > 1:
        c.ks[:] = 1 / 45                                        # the values' scales alone
    c.check()


def test_lengths_that_many_ctas_share(w4a8, cuda):
    """One long request over all SMs, beside short ones; the workspace is left as the next call expects it, and two calls give the same bits."""
    c = Case(w4a8, cuda, [20000, 3, 700], [1, 1, 2], 4, 1, 64, 64, seed=21)
    ws = torch.zeros(w4a8.attention_q8_workspace_bytes(4, w4a8.KVCache(dim=64)), dtype=torch.uint8, device=cuda)
    a, b = c.run(workspace=ws)[0], c.run(workspace=ws)[0]
    assert np.array_equal(a, b)
    o, _, reach, vmax = c.plain()
    assert (np.abs(a - o) <= c.tolerance(reach, vmax, o)[0]).all()


def test_many_requests(w4a8, cuda):
    """More requests than one launch takes."""
    R = 2500
    Case(w4a8, cuda, [1 + i % 37 for i in range(R)], [1] * R, 2, 1, 64, 16, seed=2).check()


def test_another_stream_and_an_unknown_max_q(w4a8, cuda):
    c = Case(w4a8, cuda, [300, 130], [5, 2], 4, 2, 128, 16, seed=8)
    want = c.run()[0]
    st = torch.cuda.Stream()
    assert np.array_equal(c.run(stream=st)[0], want)
    c.check(max_q=0)


def test_blocks_shared_by_requests(w4a8, cuda):
    """Two requests with a common prefix name the same blocks."""
    c = Case(w4a8, cuda, [200, 200], [1, 3], 4, 2, 128, 16, seed=9)
    c.table[1, :10] = c.table[0, :10]
    c.check()


def test_table_entry_outside_the_cache_is_reported(w4a8, cuda):
    for bad in (10 ** 6, -1):
        c = Case(w4a8, cuda, [200], [1], 4, 2, 128, 16)
        c.table[0, 3] = bad
        with pytest.raises(w4a8.W4A8Error) as e:
            c.run()
        assert e.value.code == w4a8.ERR_DEVICE and "block table" in str(e.value)
    c = Case(w4a8, cuda, [200], [1], 4, 2, 128, 16)
    c.seqs = c.seqs + 1000                                      # more tokens than the table's row holds
    with pytest.raises(w4a8.W4A8Error) as e:
        c.run()
    assert e.value.code == w4a8.ERR_DEVICE
    Case(w4a8, cuda, [200], [1], 4, 2, 128, 16).check()         # and the next call is fine


def test_blocks_past_two_to_the_31_bytes(w4a8, cuda):
    c = Case(w4a8, cuda, [150], [1], 4, 1, 128, 16, seed=13)
    want = c.check()
    blocks = 1_200_000
    far = np.array(c.table)
    dev = [torch.zeros((blocks, 1, 16, 128), dtype=torch.int8, device=cuda) for _ in range(2)] + [torch.zeros((blocks, 1), device=cuda) for _ in range(2)]
    n = len(c.ks)
    for d, a in zip(dev, (c.k, c.v, c.ks, c.vs)):
        d[blocks - n:] = to_dev(a, cuda)
    far[far >= 0] += blocks - n
    cache = w4a8.KVCache.of(*dev)
    q, out = c.q.to(cuda).contiguous(), torch.zeros((c.T, 4, 128), device=cuda)
    ws = torch.zeros(w4a8.attention_q8_workspace_bytes(4, cache), dtype=torch.uint8, device=cuda)
    w4a8.launch_attention_q8(q, 512, cache, to_dev(far, cuda), c.width, to_dev(c.cu, cuda), to_dev(c.seqs, cuda), 1, c.T, 4, out, 512, c.scale, "fp32", ws, max_q=1)
    w4a8.device_status()
    assert np.array_equal(out[:1].cpu().numpy(), want)


def test_decode_inside_a_graph(w4a8, cuda):
    """Captured once, replayed with other lengths: nothing of a call depends on what the lengths were at capture."""
    c = Case(w4a8, cuda, [300, 130, 64], [1, 1, 1], 4, 2, 128, 16, seed=10)
    dev = [to_dev(a, cuda) for a in (c.k, c.v, c.ks, c.vs)]
    cache = w4a8.KVCache.of(*dev)
    q, out = c.q.to(cuda).contiguous(), torch.zeros((c.T, 4, 128), device=cuda)
    table, cu, seqs = to_dev(c.table, cuda), to_dev(c.cu, cuda), to_dev(np.array([1, 1, 1], np.int32), cuda)
    ws = torch.zeros(w4a8.attention_q8_workspace_bytes(4, cache), dtype=torch.uint8, device=cuda)

    def call():
        w4a8.launch_attention_q8(q, 512, cache, table, c.width, cu, seqs, 3, c.T, 4, out, 512, c.scale, "fp32", ws, max_q=1)
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    seqs.copy_(to_dev(c.seqs, cuda))
    g.replay()
    w4a8.device_status()
    assert np.array_equal(out[:3].cpu().numpy(), c.run()[0])


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("vs", [0.0, 1e-25, 1e15])
@pytest.mark.parametrize("news", [[1, 1, 5], [70, 1, 90]])
def test_values_of_extreme_scale(w4a8, cuda, dtype, D, vs, news):
    """All values zero (as rows of zeros are held: scale 0, codes 0), tiny or huge: the sum of the weights is what it is without them."""
    c = Case(w4a8, cuda, [100, 17, 300], news, 8, 2, D, 16, dtype, seed=D)
    c.vs[np.isfinite(c.vs)] = vs
    if vs == 0.0:
        c.v[:] = 0
    c.check()
