"""CPU tests of the block tables' free list: what ended requests held is handed out again, once."""
import importlib

import numpy as np
import pytest
import torch

import kv_plain


@pytest.mark.parametrize("block,width,blocks,requests", [(16, 4, 12, 5), (32, 3, 7, 3), (16, 1, 4, 4)])
def test_blocks_of_ended_requests_are_free_again(w4a8, block, width, blocks, requests):
    """Random lives of requests over a pool that they need many times over: held and free blocks are all blocks at any time."""
    t = importlib.import_module(w4a8.__name__ + ".attention_block").PagedTables(requests, width, blocks, block, "cpu")
    rng, taken = np.random.default_rng(blocks), 0
    for _ in range(60):
        new = rng.integers(0, 2 * block, requests)
        new[t.kv_len.numpy() + new > width * block] = 0
        p = kv_plain.plan(t.kv_len.numpy(), new, block, t.table.numpy(), t.free.numpy()[:blocks], int(t.first), int(new.sum()))
        t.table, t.seq_len, t.status = torch.from_numpy(p["table"]), torch.from_numpy(p["seq_len"]), torch.from_numpy(p["status"])
        taken += int(p["status"][2])
        t.done()
        t.release(torch.from_numpy(rng.random(requests) < 0.4))
        held = t.table[t.table >= 0].tolist()
        assert len(held) == int(t.first) == int((-(-t.kv_len // block)).sum())
        assert sorted(held + t.free[int(t.first):blocks].tolist()) == list(range(blocks))
    assert taken > 5 * blocks


def test_nothing_ends(w4a8):
    t = importlib.import_module(w4a8.__name__ + ".attention_block").PagedTables(3, 2, 6, 16, "cpu")
    t.kv_len[:] = torch.tensor([17, 0, 3])
    t.table[0], t.table[2, 0], t.first[0] = torch.tensor([0, 1]), 2, 3
    before = [x.clone() for x in (t.kv_len, t.table, t.first, t.free[3:6])]
    t.release(torch.tensor([False, True, False]))
    assert all(torch.equal(a, b) for a, b in zip(before, (t.kv_len, t.table, t.first, t.free[3:6])))
