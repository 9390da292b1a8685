"""CPU tests: attention's arguments that have no meaning in fp32 are refused before any device work."""
import ctypes

import pytest

P = ctypes.c_void_p(4096)


@pytest.mark.parametrize("softcap,refused", [(float("inf"), True), (-0.5, True), (1e-31, True), (1e31, True), (1e-45, True), (1e-30, False), (1e30, False), (50.0, False), (0.0, False)])
def test_caps(w4a8, softcap, refused):
    """A cap that is infinite, or whose quotients leave fp32, would give rows that are not numbers.  T = 0: what is not refused has nothing to do."""
    cache = w4a8.KVCache(4096, 4096, 4096, 4096, 8, 2, 16, 64)
    rc = w4a8.lib().w4a8_attention_q8(P, 256, cache, P, 4, P, P, 1, 0, 4, P, 256, None, 0.1, 1, 0, softcap, 1, 0, P, ctypes.c_size_t(1 << 40), None)
    assert rc == (w4a8.ERR_ARG if refused else w4a8.OK)
