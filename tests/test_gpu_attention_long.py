"""GPU tests of attention over very many keys: a pool of 4096 distinct tokens, named again and again by long block tables, so that 64 bits tell the
result from the distinct ones.  Values are of one sign, so that what a sum loses with every step shows.

Tolerance: that of the attention tests (scores reach * 2^-23 * (dim / 16 + 8), weights that and 2^-18, fp16's rounding 2^-11 for 16-bit rows of prompts,
sums over the keys 2^-18, each once for numerator and denominator, and the result's own rounding).
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
OUT = {"fp32": 2.0 ** -23, "fp16": 2.0 ** -11, "bf16": 2.0 ** -8}


def long_tables(w, cuda, dtype, D, keys, requests, rows, block=64, seed=1):
    """Every request has `keys` tokens (a multiple of 4096) and `rows` queries, none of them masked; one head."""
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    blocks = 4096 // block
    k = torch.randint(-127, 128, (blocks, 1, block, D), generator=g, device=cuda, dtype=torch.int8)
    v = torch.randint(80, 128, (blocks, 1, block, D), generator=g, device=cuda, dtype=torch.int8)
    ks, vs = torch.full((blocks, 1), 0.01, device=cuda), torch.full((blocks, 1), 0.0073, device=cuda)
    cache = w.KVCache.of(k, v, ks, vs)
    width = keys // block
    table = (torch.arange(width, device=cuda, dtype=torch.int32) % blocks).repeat(requests, 1)
    T = requests * rows
    q = torch.randn((T, D), generator=g, device=cuda).to(DT[dtype])
    out, lse = torch.zeros_like(q), torch.zeros((T, 1), device=cuda)
    ws = torch.zeros(w.attention_q8_workspace_bytes(1, cache), dtype=torch.uint8, device=cuda)
    cu, seq = torch.arange(requests + 1, dtype=torch.int32, device=cuda) * rows, torch.full((requests,), keys, dtype=torch.int32, device=cuda)
    w.launch_attention_q8(q, D, cache, table, width, cu, seq, requests, T, 1, out, D, D ** -0.5, dtype, ws, causal=0, max_q=rows, lse=lse)
    w.device_status()
    kk, vv = k.double().reshape(-1, D) * float(ks[0]), v.double().reshape(-1, D) * float(vs[0])
    z = q.double() @ kk.T * D ** -0.5
    want, reach = torch.softmax(z, 1) @ vv, float((q.double().abs() @ kk.abs().T).max()) * D ** -0.5
    weight = reach * 2.0 ** -23 * (D / 16 + 8) + 2.0 ** -18 + (2.0 ** -11 if rows > 64 and dtype != "fp32" else 0.0)
    assert float(((out.double() - want).abs() - OUT[dtype] * want.abs()).max()) <= 2 * (weight + 2.0 ** -18) * float(vv.max())
    sums = torch.logsumexp(z, 1) + torch.log(torch.tensor(keys / 4096.0, dtype=torch.float64))
    assert float((lse[:, 0].double() - sums).abs().max()) <= weight + 2.0 ** -18 * (1 + float(sums.max()))


@pytest.mark.parametrize("dtype,keys", [(t, n) for t in DT for n in (32768, 36864)] + [("fp16", 1 << 20), ("bf16", 1 << 20)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_prompts_over_many_keys(w4a8, cuda, dtype, D, keys):
    """Around the length where 16-bit rows' sums move to registers, and one where the tensor core's sums would be 0.6 % off."""
    long_tables(w4a8, cuda, dtype, D, keys, 1, 140)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_so_many_tiles_that_whole_sums_are_read_out(w4a8, cuda, dtype, D):
    """Single tokens: more than 900 tiles for each of a CTA's two groups, where whole numbers would leave 32 bits."""
    long_tables(w4a8, cuda, dtype, D, 60 * 4096, 150, 1, block=128)
