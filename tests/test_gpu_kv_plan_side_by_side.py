"""A plan whose arrays lie side by side in one buffer, outputs directly behind inputs: none of them overlaps another."""
import numpy as np
import pytest
import torch

import kv_plain

pytestmark = pytest.mark.gpu


def test_arrays_side_by_side(w4a8, cuda):
    kv, new, free, table = [3, 0, 16], [2, 20, 1], [4, 7, 5, 9], np.full((3, 2), -1, np.int32)
    table[0, 0], table[2, 0] = 1, 2
    T = 23
    want = kv_plain.plan(kv, new, 16, table, free, 0, T)
    parts = {"kv": kv, "seq_len": [-9] * 3, "new": new, "cu": [-9] * 4, "free": free, "slot": [-9] * T, "first": [0], "status": [-9] * 4, "table": table.flatten().tolist(), "position": [-9] * T}
    flat = torch.tensor(sum(parts.values(), []), dtype=torch.int32, device=cuda)
    at = dict(zip(parts, flat.split([len(p) for p in parts.values()])))
    w4a8.kv_plan(at["kv"], at["new"], 3, 16, at["table"], 2, at["free"], 4, at["first"], at["seq_len"], at["cu"], at["slot"], at["position"], T, at["status"])
    w4a8.device_status()
    for k, v in want.items():
        assert np.array_equal(at[k].cpu().numpy(), v.flatten()), k
