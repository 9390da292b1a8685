"""CPU tests: caches whose rows of all heads cannot be counted in 31 bits are refused before any device work."""
import ctypes

import pytest

P = ctypes.c_void_p(4096)


@pytest.mark.parametrize("blocks,heads,block,refused", [(1 << 20, 31, 128, True), (1 << 24, 1, 128, True), ((1 << 24) - 1, 1, 128, False), (1 << 20, 16, 128, True), (1 << 20, 15, 128, False)])
def test_rows_of_all_heads(w4a8, blocks, heads, block, refused):
    """The tensor maps' row coordinate has 31 bits.  T = 0: what is not refused has nothing to do."""
    c = w4a8.KVCache(4096, 4096, 4096, 4096, blocks, heads, block, 64)
    want = w4a8.ERR_UNSUPPORTED if refused else w4a8.OK
    lib = w4a8.lib()
    assert lib.w4a8_kv_append_q8(P, P, 64 * heads, P, 0, c, 0, None) == want
    assert lib.w4a8_kv_read_q8(c, P, 4, P, P, 1, 0, P, P, 64 * heads, 0, None) == want
    assert lib.w4a8_attention_q8(P, 64 * heads, c, P, 4, P, P, 1, 0, heads, P, 64 * heads, None, 0.1, 1, 0, 0.0, 1, 0, P, ctypes.c_size_t(1 << 40), None) == want
