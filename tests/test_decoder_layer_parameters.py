"""CPU tests: parameters that a launch in the middle of a block or layer would refuse, after the stream or the cache has been changed, are refused when the block or layer is made."""
import pytest
import torch

from test_decoder_layer_refusals import D, E, H, HKV, HQ, INNER, eight, four, parts       # noqa: F401  (a fixture)


def off(t):
    """The same numbers four bytes off an aligned address."""
    raw = torch.zeros(t.numel() * t.element_size() + 4, dtype=torch.uint8)
    return raw[4:].view(t.dtype).view(t.shape) if t.element_size() <= 4 else t


def test_attention_blocks(w4a8, parts):                       # noqa: F811
    block, _ = parts
    block()
    block(rotate=w4a8.Rope.of(D, D, device="cpu"))
    for bad, why in ((dict(window=-1), "window"), (dict(softcap=-3.0), "softcap"), (dict(softcap=float("inf")), "softcap"), (dict(scale=float("nan")), "scale"),
                     (dict(rotate=w4a8.Rope.of(D, 12, device="cpu")), "rotary"), (dict(rotate=w4a8.Rope.of(D, D, variant=3, device="cpu")), "variant"),
                     (dict(rotate=w4a8.Rope.of(D, D, variant=0, device="cpu")), "weight"), (dict(wo=(off(eight(H, HQ * D)[0]), eight(H, HQ * D)[1])), "16-byte")):
        with pytest.raises((ValueError, w4a8.W4A8Error), match=why):
            block(**bad)
    assert HKV < HQ


def test_layers(w4a8, parts):                                 # noqa: F811
    _, make = parts
    make()
    for bad, why in ((dict(norm_in=w4a8.Norm.of(H, variant=0)), "norm_in"), (dict(norm_mlp=w4a8.Norm.of(H, variant=2, post_variant=1)), "norm_mlp"), (dict(norm_mlp=w4a8.Norm.of(H, variant=5)), "variant"),
                     (dict(norm_mlp=w4a8.Norm.of(H, variant=2, eps=-1.0)), "eps"), (dict(router=w4a8.Router.of(E, 9)), "experts"), (dict(router=w4a8.Router.of(E, 2, groups=3)), "groups"),
                     (dict(act=2), "act"), (dict(inner=48, gate_up=four(E * 96, H), down=(torch.zeros(E * H, 24, dtype=torch.uint8), torch.zeros(E * H * 48 // 32))), "multiples of 32"),
                     (dict(gate_up=(off(four(E * 2 * INNER, H)[0]), four(E * 2 * INNER, H)[1])), "16-byte"), (dict(down=(four(E * H, INNER)[0], off(four(E * H, INNER)[1]))), "16-byte"),
                     (dict(router_w=(off(eight(E, H)[0]), eight(E, H)[1])), "16-byte")):
        with pytest.raises((ValueError, w4a8.W4A8Error), match=why):
            make(**bad)
