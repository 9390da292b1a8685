"""Frequencies of rotary positions (w4a8_rope_table) against fifty decimal digits; no GPU."""
import math
from decimal import Decimal, getcontext

import pytest

getcontext().prec = 50
PI = Decimal("3.14159265358979323846264338327950288419716939937510")


def _plain(rotary, base, i):
    return (Decimal(base).ln() * Decimal(-2 * i) / Decimal(rotary)).exp()


def _close(w4a8, rotary, want, base=10000.0, scaling="none", **more):
    turns, magnitude = w4a8.rope_table(rotary, base, scaling, **more)
    assert len(turns) == rotary // 2
    for i, t in enumerate(turns):
        # long double: the exponent's rounding times ln(base), the power's, two divisions: 24 * 2^-64 of at most a sixth of a turn; the ramps' some more
        assert abs(Decimal(t) - want(i) / (2 * PI) * 2 ** 64) <= 40, (i, t)
    return magnitude


@pytest.mark.parametrize("rotary,base", [(128, 10000.0), (64, 500000.0), (2, 10000.0), (24, 1e6), (1024, 10000.0)])
def test_plain_frequencies(w4a8, rotary, base):
    assert _close(w4a8, rotary, lambda i: _plain(rotary, base, i), base) == 1.0


def test_scaled_frequencies(w4a8):
    R, b, s = 128, 500000.0, Decimal(8)
    assert _close(w4a8, R, lambda i: _plain(R, b, i) / s, b, "linear", factor=8.0) == 1.0
    stretched = (s.ln() * Decimal(R) / (R - 2)).exp() * Decimal(b)
    _close(w4a8, R, lambda i: (stretched.ln() * Decimal(-2 * i) / R).exp(), b, "ntk", factor=8.0)
    d = [1.0 + 0.25 * i for i in range(R // 2)]
    _close(w4a8, R, lambda i: _plain(R, b, i) / Decimal(d[i]), b, "divisors", divisors=d)

    def bands(i):
        f = _plain(R, b, i)
        ramp = min(Decimal(1), max(Decimal(0), (8192 * f / (2 * PI) - 1) / 3))
        return f * (ramp + (1 - ramp) / s)
    _close(w4a8, R, bands, b, "bands", factor=8.0, original=8192.0)

    def yarn(i):
        at = lambda n: R * (Decimal(4096) / (n * 2 * PI)).ln() / (2 * Decimal(10000).ln())
        lo, hi = max(0, math.floor(at(32))), min(R - 1, math.ceil(at(1)))
        ramp = min(Decimal(1), max(Decimal(0), Decimal(i - lo) / (hi - lo)))
        return _plain(R, 10000.0, i) * (1 - ramp + ramp / s)
    m = _close(w4a8, R, yarn, 10000.0, "yarn", factor=8.0, original=4096.0)
    assert abs(m - (0.1 * math.log(8.0) + 1)) < 1e-7


def test_refusals(w4a8):
    for args in [(3,), (-2,), (2048,), (64, 0.0), (64, float("nan")), (64, 10000.0, "linear", 0.0), (64, 10000.0, "yarn", 8.0, 0.0), (64, 10000.0, "bands", 8.0, 4096.0, 4.0, 1.0),
                 (64, 1.0, "yarn", 8.0, 4096.0)]:
        with pytest.raises(w4a8.W4A8Error) as e:
            w4a8.rope_table(*args)
        assert e.value.code == w4a8.ERR_ARG
    with pytest.raises(w4a8.W4A8Error):
        w4a8.rope_table(4, 10000.0, "divisors", divisors=[1.0, 0.0])
    with pytest.raises(w4a8.W4A8Error):
        w4a8.rope_table(4, 10000.0, "divisors")
    with pytest.raises(ValueError):
        w4a8.rope_table(4, 10000.0, "divisors", divisors=[1.0])
    assert w4a8.rope_table(0) == ([], 1.0)
