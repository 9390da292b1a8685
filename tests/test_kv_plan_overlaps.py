"""CPU tests: a plan's outputs that lie in its inputs are refused before any device work, whichever and however far."""
import ctypes

import pytest

R, T, WIDTH, FREE = 5, 7, 4, 6
SIZES = {"kv_len": R, "new_len": R, "free_blocks": FREE, "first_free": 1, "seq_len": R, "cu_new": R + 1, "slot": T, "position": T, "status": 4, "block_table": R * WIDTH}
INPUTS = ("kv_len", "new_len", "free_blocks", "first_free")


def call(w, **places):
    at = {name: 4096 * (i + 1) for i, name in enumerate(SIZES)}
    at.update(places)
    a = {k: ctypes.c_void_p(v) for k, v in at.items()}
    return w.lib().w4a8_kv_plan(a["kv_len"], a["new_len"], R, 16, a["block_table"], WIDTH, a["free_blocks"], FREE, a["first_free"], a["seq_len"], a["cu_new"], a["slot"],
                                a["position"], T, a["status"], None), at


@pytest.mark.parametrize("i", INPUTS)
@pytest.mark.parametrize("o", [n for n in SIZES if n not in INPUTS])
def test_outputs_in_inputs(w4a8, i, o):
    base = call(w4a8)[1][i]
    for place in {base, base + 4 * (SIZES[i] - 1), base - 4 * (SIZES[o] - 1)}:            # the same, the last element of one the first of the other
        assert call(w4a8, **{o: place})[0] == w4a8.ERR_ARG
        text = w4a8.lib().w4a8_last_error().decode()
        assert o in text and i in text
