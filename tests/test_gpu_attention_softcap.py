"""GPU tests of capped scores: cap * tanh(score / cap) is as exact as the score it is made of, for any cap and beside values of any scale.

With a window of one token a row's lse is its one capped score.  Its tolerance: the score's own, reach * 2^-23 * (dim / 16 + 8), which tanh does not
widen; a relative 2^-20 for the quotient by the cap, tanh and the product with the cap (each at most a few units of 2^-23); and 2^-18 of
1 + |lse| for two exponentials (2^-22 each), up to four roundings of their arguments (numbers below 16: 2^-21 each) and the logarithm.
"""
import numpy as np
import pytest

from test_gpu_attention_q8 import Case
from test_gpu_attention_scales import compare, scaled

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("news", [[1, 2, 5], [70, 100, 65]])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("cap", [0.5, 5.0, 50.0, 1000.0, 1e5, 1e12])
@pytest.mark.parametrize("scales", [(1 / 45,), (0.0,), (1e-25, 1e10)])
def test_one_score_a_row(w4a8, cuda, news, D, cap, scales):
    for sharp in (0.01, 0.3):
        c = scaled(Case(w4a8, cuda, [300, 129, 70], news, 4, 2, D, 16, window=1, softcap=cap, sharp=sharp, seed=D), scales)
        _, lse = c.run()
        _, l, reach, _ = c.plain()
        tol = reach * 2.0 ** -23 * (D / 16 + 8) + 2.0 ** -20 * np.abs(l) + 2.0 ** -18 * (1 + np.abs(l))
        assert (np.abs(lse - l) <= tol).all(), float((np.abs(lse - l) - tol).max())


@pytest.mark.parametrize("news", [[1, 2, 5], [70, 100, 65]])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("cap", [5.0, 50.0, 1e5])
@pytest.mark.parametrize("scales", [(1 / 45, 1e-6), (0.0, 1 / 45), (0.0, 1e-25, 1e10)])
def test_capped_beside_values_of_any_scale(w4a8, cuda, news, dtype, cap, scales):
    compare(scaled(Case(w4a8, cuda, [300, 129, 70], news, 8, 2, 128, 16, dtype, softcap=cap, sharp=3.0, seed=9), scales))
