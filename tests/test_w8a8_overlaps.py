"""CPU tests: what w4a8_linear_w8a8 writes besides Y, the rows' codes and scales, overlaps none of what it reads."""
import ctypes

import pytest
import torch

GPU = torch.cuda.is_available()      # the pointers are made up: calls that are allowed get as far as the device check, without a device
BASE = 1 << 20
S, N, K = 2, 40, 64


def call(w4a8, rows=S, skip=0, **at):
    p = dict(x=BASE, xq=BASE << 1, xs=BASE << 2, wq=BASE << 3, ws=BASE << 4, bias=BASE << 5, Y=BASE << 6) | at
    P = lambda n: ctypes.c_void_p(p[n])
    return w4a8.lib().w4a8_linear_w8a8(P("x"), K, P("xq"), P("xs"), P("wq"), P("ws"), P("bias"), P("Y"), N, rows, N, K, 0, 0, skip, None)


@pytest.mark.parametrize("rows", [1, 2, 5])
@pytest.mark.parametrize("at,what", [
    (dict(xq=BASE << 3), b"xq overlaps wq"), (dict(xq=(BASE << 3) + N * K - 16), b"xq overlaps wq"), (dict(xq=BASE << 4), b"xq overlaps ws"), (dict(xq=BASE << 5), b"xq overlaps bias"),
    (dict(xs=BASE << 4), b"xs overlaps ws"), (dict(xs=(BASE << 4) + 4 * N - 4), b"xs overlaps ws"), (dict(xs=BASE << 5), b"xs overlaps bias"), (dict(xs=(BASE << 3) + 64), b"xs overlaps wq"),
    (dict(xs=BASE << 1), b"xs overlaps xq"), (dict(xq=BASE), b"xq overlaps x"), (dict(xs=BASE + 16), b"xs overlaps x")])
def test_codes_and_scales_in_the_place_of_an_input(w4a8, rows, at, what):
    assert call(w4a8, rows, **at) == w4a8.ERR_ARG and what in w4a8.lib().w4a8_last_error()


@pytest.mark.skipif(GPU, reason="made-up pointers")
def test_rows_that_are_quantized_already_may_lie_anywhere(w4a8):
    for at in (dict(xs=BASE << 4), dict(xq=BASE << 3), {}):
        assert call(w4a8, skip=1, **at) not in (w4a8.ERR_ARG, w4a8.ERR_ALIGN)
    assert call(w4a8) not in (w4a8.ERR_ARG, w4a8.ERR_ALIGN)
    assert call(w4a8, xq=(BASE << 3) + N * K, xs=(BASE << 4) + 4 * N) not in (w4a8.ERR_ARG, w4a8.ERR_ALIGN)      # side by side
