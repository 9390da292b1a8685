"""CPU tests: what the 8-bit KV cache's entry points refuse before any device work, and the plain plan they are compared with."""
import ctypes

import numpy as np
import pytest

import kv_plain

P = ctypes.c_void_p(4096)


def cache(w, **kw):
    f = dict(k=4096, v=4096, k_scale=4096, v_scale=4096, num_blocks=8, heads=2, block=16, dim=64)
    f.update(kw)
    return w.KVCache(*(f[n] for n, _ in w.KVCache._fields_))


@pytest.mark.parametrize("change,code", [
    (dict(dim=80), "ARG"), (dict(block=24), "ARG"), (dict(block=256), "ARG"), (dict(heads=0), "ARG"), (dict(num_blocks=0), "ARG"), (dict(k=None), "ARG"),
    (dict(v_scale=None), "ARG"), (dict(v=4104), "ALIGN"), (dict(num_blocks=1 << 28), "UNSUPPORTED"), (dict(num_blocks=1 << 20, heads=1000, block=128), "UNSUPPORTED"),
])
def test_caches_that_are_refused(w4a8, change, code):
    lib, c = w4a8.lib(), cache(w4a8, **change)
    want = getattr(w4a8, "ERR_" + code)
    ws = ctypes.c_size_t(1 << 40)
    assert lib.w4a8_kv_append_q8(P, P, 128, P, 3, c, 0, None) == want
    assert lib.w4a8_kv_read_q8(c, P, 4, P, P, 1, 3, P, P, 128, 0, None) == want
    assert lib.w4a8_attention_q8(P, 256, c, P, 4, P, P, 1, 1, 4, P, 256, None, 0.1, 1, 0, 0.0, 1, 0, P, ws, None) == want
    assert lib.w4a8_last_error() != b""


def test_rows_that_are_refused(w4a8):
    lib, c = w4a8.lib(), cache(w4a8)
    odd = ctypes.c_void_p(4104)
    assert lib.w4a8_kv_append_q8(P, P, 128, P, 3, c, 3, None) == w4a8.ERR_ARG              # dtype
    assert lib.w4a8_kv_append_q8(P, P, 127, P, 3, c, 0, None) == w4a8.ERR_ARG              # rows overlap
    assert lib.w4a8_kv_append_q8(P, P, 132, P, 3, c, 1, None) == w4a8.ERR_ALIGN            # 264-byte rows
    assert lib.w4a8_kv_append_q8(P, odd, 128, P, 3, c, 0, None) == w4a8.ERR_ALIGN
    assert lib.w4a8_kv_append_q8(P, P, 128, None, 3, c, 0, None) == w4a8.ERR_ARG
    assert lib.w4a8_kv_append_q8(P, P, 128, P, -1, c, 0, None) == w4a8.ERR_ARG
    assert lib.w4a8_kv_append_q8(None, None, 128, None, 0, c, 0, None) == w4a8.OK          # nothing to write
    assert lib.w4a8_kv_read_q8(c, P, 4, None, P, 1, 3, P, P, 128, 0, None) == w4a8.ERR_ARG
    assert lib.w4a8_kv_read_q8(c, P, 4, P, P, -1, 3, P, P, 128, 0, None) == w4a8.ERR_ARG
    assert lib.w4a8_kv_read_q8(c, P, 4, P, P, 1, 0, None, None, 128, 0, None) == w4a8.OK


def test_attention_arguments_that_are_refused(w4a8):
    lib, c = w4a8.lib(), cache(w4a8)
    big = ctypes.c_size_t(1 << 40)

    def call(q=P, ldq=256, heads=4, scale=0.1, window=0, softcap=0.0, dtype=0, ws=P, n=big, R=1, T=1, table=P, max_q=1, width=4):
        return lib.w4a8_attention_q8(q, ldq, c, table, width, P, P, R, T, heads, P, 256, None, scale, 1, window, softcap, max_q, dtype, ws, n, None)
    assert call(heads=3) == w4a8.ERR_ARG                                                  # not a multiple of the kv heads
    assert call(heads=0) == w4a8.ERR_ARG
    assert call(window=-1) == w4a8.ERR_ARG
    assert call(softcap=-1.0) == w4a8.ERR_ARG
    assert call(softcap=float("nan")) == w4a8.ERR_ARG
    assert call(scale=float("nan")) == w4a8.ERR_ARG
    assert call(dtype=4) == w4a8.ERR_ARG
    assert call(ldq=255) == w4a8.ERR_ARG
    assert call(ldq=258) == w4a8.ERR_ALIGN
    assert call(q=ctypes.c_void_p(4100)) == w4a8.ERR_ALIGN
    assert call(table=None) == w4a8.ERR_ARG
    assert call(max_q=-1) == w4a8.ERR_ARG
    assert call(ws=None) == w4a8.ERR_WORKSPACE
    assert call(n=ctypes.c_size_t(64)) == w4a8.ERR_WORKSPACE and b"workspace" in lib.w4a8_last_error()
    assert call(ws=ctypes.c_void_p(4096 + 16)) == w4a8.ERR_ALIGN
    assert call(R=0) == w4a8.OK and call(T=0) == w4a8.OK                                  # nothing to do
    assert w4a8.attention_q8_workspace_bytes(0, c) == 0
    assert w4a8.attention_q8_workspace_bytes(4, c, 1, 1) > 0


def test_plan_arguments_that_are_refused(w4a8):
    lib = w4a8.lib()

    def call(R=2, block=16, width=4, num_free=4, T=3, kv=P, seq=ctypes.c_void_p(8192), free=P, slot=P, status=P):
        return lib.w4a8_kv_plan(kv, P, R, block, P, width, free, num_free, P, seq, P, slot, None, T, status, None)
    assert call(R=-1) == w4a8.ERR_ARG
    assert call(block=17) == w4a8.ERR_ARG
    assert call(num_free=-1) == w4a8.ERR_ARG
    assert call(seq=P) == w4a8.ERR_ARG                                                    # seq_len must not be kv_len
    assert call(free=None) == w4a8.ERR_ARG
    assert call(slot=None) == w4a8.ERR_ARG
    assert call(status=None) == w4a8.ERR_ARG
    assert call(R=20000) == w4a8.ERR_UNSUPPORTED


def test_cache_tensors_that_do_not_fit_together(w4a8):
    import torch
    k, s = torch.zeros((3, 2, 16, 64), dtype=torch.int8), torch.zeros((3, 2))
    c = w4a8.KVCache.of(k, k.clone(), s, s.clone())
    assert (c.num_blocks, c.heads, c.block, c.dim) == (3, 2, 16, 64)
    for bad in ((k, k[:2].clone(), s, s), (k, k, s, torch.zeros((3, 3))), (k, k, s.half(), s), (k.float(), k.float(), s, s), (k.transpose(2, 3), k, s, s)):
        with pytest.raises(ValueError):
            w4a8.KVCache.of(*bad)


def test_plain_plan_by_hand():
    """Three requests over a list of three free blocks: the second needs two and gets them, the third's one is the last, the fourth goes without."""
    table = np.full((4, 3), -1, np.int32)
    table[0, 0] = 9
    got = kv_plain.plan([15, 0, 0, 0], [1, 20, 1, 1], 16, table, [4, 7, 5], 0, 24)
    assert got["table"][0].tolist() == [9, -1, -1] and got["table"][1].tolist() == [4, 7, -1] and got["table"][2, 0] == 5 and got["table"][3, 0] == -1
    assert got["seq_len"].tolist() == [16, 20, 1, 0] and got["cu"].tolist() == [0, 1, 21, 22, 23]
    assert got["slot"][0] == 9 * 16 + 15 and got["slot"][1] == 64 and got["slot"][20] == 7 * 16 + 3 and got["slot"][21] == 80 and got["slot"][22:].tolist() == [-1, -1]
    assert got["status"].tolist() == [3, 1, 3, 22]
