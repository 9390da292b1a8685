"""CPU tests with stand-ins: structs, matrices and rows on another GPU than the launch's, or than their block's, are refused; a kernel would follow their
pointers to a fault."""
import importlib

import pytest
import torch

from test_decoder_layer_refusals import D, E, H, HKV, HQ, INNER, eight, four, parts       # noqa: F401  (a fixture)

BASE = 1 << 20


class On:
    """What the package looks at of an fp32 vector on GPU `gpu`."""
    dtype, is_cuda = torch.float32, True

    def __init__(self, n, gpu):
        self.n, self.gpu = n, gpu

    def numel(self):
        return self.n

    def is_contiguous(self):
        return True

    def get_device(self):
        return self.gpu

    def data_ptr(self):
        return BASE

    def dim(self):
        return 1

    @property
    def shape(self):
        return (self.n,)

    def stride(self, _):
        return 1


def test_tensors_of_one_struct_lie_on_one_gpu(w4a8):
    for make in (lambda: w4a8.Norm.of(64, On(64, 0), post_weight=On(64, 1), post_variant=0), lambda: w4a8.Norm.of(64, On(64, 0), gate=On(64, 1)),
                 lambda: w4a8.Rope.of(64, 64, q_weight=On(64, 0), k_weight=On(64, 1), variant=0, device="cpu"), lambda: w4a8.Rope.of(64, 64, q_weight=On(64, 0), k_weight=On(64, 0), variant=0, device="cpu")):
        with pytest.raises(ValueError, match="not on one GPU"):
            make()
    assert w4a8.Norm.of(64, On(64, 1), gate=On(64, 1))._gpu == 1 and w4a8.Norm.of(64, variant=2)._gpu is None and w4a8.Router.of(64, 4, bias=On(64, 3))._gpu == 3
    assert w4a8.Rope.of(64, 0, q_weight=On(64, 2), k_weight=On(64, 2), variant=0, device="cpu")._gpu == 2            # no table


def test_structs_on_another_gpu_than_the_current_one(w4a8):
    """The calls have no rows: nothing is launched, whatever they are asked."""
    b = w4a8._binding()
    norm, router, rope = w4a8.Norm.of(64, On(64, 1)), w4a8.Router.of(64, 4, bias=On(64, 1)), w4a8.Rope.of(64, 0, q_weight=On(64, 1), k_weight=On(64, 1), variant=0, device="cpu")
    calls = [lambda: w4a8.launch_add_norm(norm, BASE, None, 0, stream=0), lambda: w4a8.launch_moe_route(router, BASE, 64, 0, BASE, BASE, stream=0),
             lambda: w4a8.launch_rope_qk(rope, BASE, 64, 1, BASE, 64, 1, BASE, 0, stream=0)]
    try:
        b.streams(lambda: 0, lambda device: 0, 2, torch.Tensor)
        for call in calls:
            with pytest.raises(ValueError, match="on GPU 1, the current one is 0"):
                call()
        w4a8.launch_add_norm(w4a8.Norm.of(64, variant=2), BASE, None, 0, stream=0)       # nothing to follow
        b.streams(lambda: 1, lambda device: 0, 2, torch.Tensor)
        for call in calls:
            call()
    finally:
        w4a8._native = None                                  # bound anew with torch's own functions


def test_blocks_of_parts_on_other_gpus(w4a8, parts):                                     # noqa: F811
    block, make = parts
    with pytest.raises(ValueError, match="norm_in"):
        make(norm_in=w4a8.Norm.of(H, On(H, 1)))
    with pytest.raises(ValueError, match="norm_mlp"):
        make(norm_mlp=w4a8.Norm.of(H, On(H, 0)))
    with pytest.raises(ValueError, match="router"):
        make(router=w4a8.Router.of(E, 2, bias=On(E, 1)))
    with pytest.raises(ValueError, match="rotate"):
        block(rotate=w4a8.Rope.of(D, 0, q_weight=On(D, 1), k_weight=On(D, 1), variant=0, device="cpu"))
    away = lambda m: tuple(x.to("meta") for x in m)
    for bad in (dict(wqkv=away(four((HQ + 2 * HKV) * D, H))), dict(wo=away(eight(H, HQ * D))), dict(wo=(eight(H, HQ * D)[0], eight(H, HQ * D)[1].to("meta")))):
        with pytest.raises(ValueError, match="on cpu, as the tables"):
            block(**bad)


class Rows:
    """What a block looks at of its rows, on its own GPU."""
    dtype, is_cuda = torch.float32, True

    def __init__(self, n, device):
        self.shape, self.device = (n, H), device

    def dim(self):
        return 2

    def is_contiguous(self):
        return True


def test_rows_on_another_gpu_than_the_current_one(w4a8, parts, monkeypatch):             # noqa: F811
    block = parts[0]()
    gpu = torch.device("cuda", 1)

    class Buffer:
        device = gpu
    block.qkv = Buffer()                                     # a block of GPU 1
    block.tables.slot = torch.zeros(4, dtype=torch.int32)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    with pytest.raises(ValueError, match="not the current GPU"):
        block._check(Rows(4, gpu))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    block._check(Rows(4, gpu))
    assert INNER and HKV
