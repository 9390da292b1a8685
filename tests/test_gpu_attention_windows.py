"""GPU tests of windows as wide as their type allows, with requests that have more rows than tokens."""
import numpy as np
import pytest

from test_gpu_attention_q8 import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 4, 2 ** 30])
@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("D,seqs,news", [(64, [3, 5, 200], [7, 1, 2]), (128, [3, 40, 5], [9, 2, 70]), (256, [3], [100]), (128, [90, 20], [90, 300])])
def test_window_of_everything(w4a8, cuda, window, causal, D, seqs, news):
    c = Case(w4a8, cuda, seqs, news, 4, 2, D, 16, causal=causal, window=window, seed=D)
    got = c.run()[0]
    c.kw["window"] = 0                                           # no window is as wide, and the plain form's positions have 32 bits too
    o, _, reach, vmax = c.plain()
    assert (np.abs(got - o) <= c.tolerance(reach, vmax, o)[0]).all()
