"""CPU tests: what the attention block's Python module refuses before any launch, because its launches take plain pointers."""
import importlib

import pytest
import torch

HIDDEN, HQ, HKV, D, ROWS = 256, 6, 2, 64, 32


def weights(rows, k):
    return torch.zeros((rows, k // 2), dtype=torch.uint8), torch.zeros((rows, k // 32))


@pytest.fixture()
def block(w4a8):
    mod = importlib.import_module(w4a8.__name__ + ".attention_block")
    tables = mod.PagedTables(3, 4, 8, 16, "cpu")
    return mod, tables, mod.AttentionBlock(weights((HQ + 2 * HKV) * D, HIDDEN), weights(HIDDEN, HQ * D), HIDDEN, HQ, HKV, D, tables, ROWS)


@pytest.mark.parametrize("planned,shape,kw,why", [
    (40, (40, HIDDEN), {}, "room for 32"), (8, (9, HIDDEN), {}, "planned for 8"), (0, (3, HIDDEN), {}, "planned for 0"), (8, (8, HIDDEN - 32), {}, "rows of 256"),
    (8, (8 * HIDDEN,), {}, "rows of 256"), (8, (8, HIDDEN), dict(dtype=torch.float16), "fp32"), (8, (8, HIDDEN), {}, "on cpu"),
])
def test_rows_that_do_not_fit(block, planned, shape, kw, why):
    """More rows than the buffers or the plan have, and rows that are something else."""
    _, tables, layer = block
    tables.slot = torch.zeros(planned, dtype=torch.int32)
    with pytest.raises(ValueError, match=why):
        layer(torch.zeros(shape, **kw))


def test_rows_that_are_not_contiguous(block):
    _, tables, layer = block
    tables.slot = torch.zeros(8, dtype=torch.int32)
    with pytest.raises(ValueError, match="contiguous"):
        layer(torch.zeros(8, 2 * HIDDEN)[:, :HIDDEN])


def test_before_the_first_step(block):
    with pytest.raises(ValueError, match="planned for 0"):
        block[2](torch.zeros(1, HIDDEN))


@pytest.mark.parametrize("bad", [torch.zeros(3, dtype=torch.int64), torch.zeros(2, dtype=torch.int32), torch.zeros(6, dtype=torch.int32)[::2]])
def test_lengths_that_do_not_fit(block, bad):
    with pytest.raises(ValueError, match="3 int32 numbers"):
        block[1].step(bad, 4)


def test_weights_that_do_not_fit(block):
    mod, tables, _ = block
    good = weights((HQ + 2 * HKV) * D, HIDDEN), weights(HIDDEN, HQ * D)
    for bad in ((weights(HQ * D, HIDDEN), good[1]), (good[0], weights(HIDDEN, HIDDEN)), ((good[0][0], good[0][1].half()), good[1])):
        with pytest.raises(ValueError, match="packed int4"):
            mod.AttentionBlock(*bad, HIDDEN, HQ, HKV, D, tables, ROWS)
