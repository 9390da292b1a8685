"""GPU tests of attention over caches whose value scales lie far apart, or are no numbers, in one request.

The tolerance is that of the attention tests (scores, weights, sums over the keys), taken with the largest value that the ROW sees, not with the
largest of the cache; results below the smallest normal number of their type are off by one unit of it more.
"""
import numpy as np
import pytest

from test_gpu_attention_q8 import Case

pytestmark = pytest.mark.gpu
SCALES = {
    "zero beside ordinary": (0.0, 1 / 45), "zero and subnormal beside ordinary": (0.0, 1e-40, 1 / 45), "zero beside small": (0.0, 1e-8), "all small": (1e-36,),
    "all subnormal": (1e-40,), "all large": (1e25,), "all larger": (1e30,), "all as large as they get": (1e36,), "zero beside large": (0.0, 1e36),
    "small beside large": (1e-36, 1e36), "subnormal, ordinary, large": (1e-40, 1.0, 1e36), "ascending": (1e-30, 1e-20, 1e-10, 1.0, 1e10, 1e20),
    "descending": (1e20, 1e10, 1.0, 1e-10, 1e-20, 1e-30),
}


def scaled(c, pattern):
    """Block i of every request has the pattern's i-th scale (codes of zero where it is zero, as the write leaves them)."""
    for r, n in enumerate(c.seqs):
        for i in range(-(-int(n) // c.k.shape[2])):
            b = c.table[r, i]
            c.vs[b] = pattern[i % len(pattern)]
            if pattern[i % len(pattern)] == 0.0:
                c.v[b] = 0
    return c


def widest(c):
    """The largest magnitude of a value that each row sees."""
    out, block = np.zeros(int(c.cu[-1])), c.k.shape[2]
    for r, n in enumerate(c.news):
        L = int(c.seqs[r])
        amax = np.array([np.abs(c.v[c.table[r, j // block], :, j % block].astype(np.float64) * c.vs[c.table[r, j // block], :, None].astype(np.float64)).max() for j in range(L)])
        for i in range(n):
            p = L - n + i
            lo, hi = max(0, p - c.kw["window"] + 1) if c.kw["window"] else 0, p + 1 if c.kw["causal"] else L
            out[c.cu[r] + i] = amax[lo:hi].max() if hi > lo else 0.0
    return out[:, None, None]


def compare(c):
    got, lse = c.run()
    o, l, reach, _ = c.plain()
    tol, tol_l = c.tolerance(reach, widest(c), o)
    assert (np.abs(got - o) <= tol + {"fp32": 2.0 ** -149, "fp16": 2.0 ** -24, "bf16": 2.0 ** -133}[c.dtype]).all()
    assert (np.abs(lse - l) <= tol_l * (1 + np.abs(l))).all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("name", list(SCALES))
@pytest.mark.parametrize("D,news", [(64, [1, 1, 5]), (128, [1, 2, 3]), (256, [1, 1, 2])])
def test_scales_far_apart(w4a8, cuda, dtype, name, D, news):
    """Requests of few rows."""
    for window in (0, 40):
        compare(scaled(Case(w4a8, cuda, [100, 17, 300], news, 8, 2, D, 16, dtype, window=window, seed=D), SCALES[name]))


@pytest.mark.parametrize("D", [64, 128])
def test_parts_of_a_long_request(w4a8, cuda, D):
    """Partial results that are joined have references of their own kind: zeros and large values by stretches of 4096 tokens."""
    c = Case(w4a8, cuda, [20000], [1], 4, 1, D, 64, seed=5)
    compare(scaled(c, (0.0,) * 64 + (1e36,) * 64 + (1e-36,) * 64 + (1.0,) * 64))


def not_a_number(w4a8, cuda, dtype, bad, D, news):
    """Rows that see the block are not numbers (an infinity is written as codes of zero with an infinite scale), those before it are as without it."""
    c = Case(w4a8, cuda, [64 + news], [news], 4, 2, D, 16, dtype, seed=3)
    b = c.table[0, 4 + (news - 1) // 16]                       # the request's last block
    first = (news - 1) // 16 * 16                              # the first query that sees it
    side = c.vs if bad[0] == "v" else c.ks
    want = c.run()[0]
    side[b] = np.nan if "nan" in bad else np.inf
    if bad == "v inf":
        c.v[b] = 0
    got, lse = c.run()
    assert np.isnan(got[first:]).all()
    assert np.array_equal(got[:first], want[:first]) and np.isfinite(lse[:first]).all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("bad", ["v nan", "v inf", "k nan"])
@pytest.mark.parametrize("D,news", [(64, 3), (128, 5), (256, 2)])
def test_scale_that_is_not_a_number(w4a8, cuda, dtype, bad, D, news):
    not_a_number(w4a8, cuda, dtype, bad, D, news)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("name", list(SCALES))
@pytest.mark.parametrize("D", [64, 128, 256])
def test_scales_far_apart_in_prompts(w4a8, cuda, dtype, name, D):
    """70 and 90 rows are tiles of rows, the three rows between them stream."""
    for window in (0, 40):
        compare(scaled(Case(w4a8, cuda, [100, 17, 300], [70, 3, 90], 8, 2, D, 16, dtype, window=window, seed=D), SCALES[name]))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("bad", ["v nan", "v inf", "k nan"])
@pytest.mark.parametrize("D,news", [(64, 100), (128, 100), (256, 70)])
def test_scale_that_is_not_a_number_in_prompts(w4a8, cuda, dtype, bad, D, news):
    not_a_number(w4a8, cuda, dtype, bad, D, news)
