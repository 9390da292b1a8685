"""CPU tests: what the attention block and the decoder layer refuse of 8-bit weights, ropes and norms before any launch."""
import importlib

import pytest
import torch

H, HQ, HKV, D, ROWS, E, INNER = 256, 4, 2, 64, 32, 8, 64


def four(n, k):
    return torch.zeros((n, k // 2), dtype=torch.uint8), torch.zeros((n, k // 32))


def eight(n, k):
    return torch.zeros((n, k), dtype=torch.int8), torch.zeros(n)


@pytest.fixture()
def parts(w4a8):
    mod, layer = (importlib.import_module(w4a8.__name__ + "." + m) for m in ("attention_block", "decoder_layer"))
    tables = mod.PagedTables(3, 4, 8, 16, "cpu")
    block = lambda **k: mod.AttentionBlock(**({"wqkv": four((HQ + 2 * HKV) * D, H), "wo": eight(H, HQ * D), "hidden": H, "heads_q": HQ, "heads": HKV, "dim": D, "tables": tables, "max_rows": ROWS} | k))
    n = w4a8.Norm.of(H, variant=2)
    make = lambda **k: layer.DecoderLayer(**({"attention": block(), "norm_in": n, "norm_mlp": n, "router": w4a8.Router.of(E, 2), "router_w": eight(E, H), "gate_up": four(E * 2 * INNER, H),
                                              "down": four(E * H, INNER), "inner": INNER} | k))
    return block, make


def test_eight_bit_projections(parts):
    block, _ = parts
    assert block().wide_o and not block().wide_qkv
    for bad in ((torch.zeros((H, HQ * D), dtype=torch.int8), torch.zeros(H, 1).half()), (torch.zeros((H, HQ * D), dtype=torch.int8), torch.zeros(H // 2)), (torch.zeros((H, HQ * D), dtype=torch.uint8), torch.zeros(H))):
        with pytest.raises(ValueError, match="packed int4"):
            block(wo=bad)


def test_ropes_of_other_heads(w4a8, parts):
    with pytest.raises(ValueError, match="128 elements"):
        parts[0](rotate=w4a8.Rope.of(128, 128, device="cpu"))


def test_layers(w4a8, parts):
    _, make = parts
    layer = make()
    for bad, why in ((dict(norm_in=w4a8.Norm.of(H + 32, variant=2)), "norm_in"), (dict(norm_mlp=w4a8.Norm.of(H, variant=2, dtype="bf16")), "norm_mlp"), (dict(router_w=four(E, H)), "int8"),
                     (dict(router_w=eight(E + 1, H)), "router_w"), (dict(gate_up=four(E * INNER, H)), "gate_up"), (dict(down=four(E * H, 2 * INNER)), "down"), (dict(scale_dtype=1), "gate_up")):
        with pytest.raises(ValueError, match=why):
            make(**bad)
    for h, why in ((torch.zeros(4, H + 32), "h:"), (torch.zeros(4, H).half(), "h:"), (torch.zeros(4, 2 * H)[:, :H], "h:"), (torch.zeros(ROWS + 1, H), "room for")):
        with pytest.raises(ValueError, match=why):
            layer(h)
    with pytest.raises(ValueError, match="not the current GPU"):
        layer(torch.zeros(4, H))                             # a layer in host memory
    meta = lambda n, k: tuple(x.to("meta") for x in four(n, k))
    for bad in (dict(gate_up=meta(E * 2 * INNER, H)), dict(down=meta(E * H, INNER)), dict(router_w=tuple(x.to("meta") for x in eight(E, H)))):
        with pytest.raises(ValueError, match="on cpu, as the attention"):
            make(**bad)
    with pytest.raises(ValueError, match="y:"):
        layer(torch.zeros(4, H), torch.zeros(5, H))
