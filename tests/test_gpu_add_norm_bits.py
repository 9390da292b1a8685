"""How far a row's outputs may depend on how many rows a call has (w4a8_add_norm): not at all, but for a factor r on the border between two fp32 numbers, which
may be either of the two."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def border(ss, K, up):
    """An eps with which 1 / sqrt(ss / K + eps) is, to the last bits of fp64, halfway between two fp32 numbers."""
    mean = ss / K
    r = float(torch.tensor(1.0 / math.sqrt(up * mean), dtype=torch.float32))
    step = 2.0 ** (math.frexp(r)[1] - 24)
    middle = r + step / 2
    return 1.0 / (middle * middle) - mean


# one row and many: 8 elements a thread and 16, a CTA a row and a warp a row
@pytest.mark.parametrize("K,S", [(5120, 900), (3840, 700), (8192, 400), (256, 700), (512, 601), (480, 1200)])
@pytest.mark.parametrize("dtype,post", [("fp32", False), ("fp32", True), ("bf16", False)])
def test_factors_on_a_border(w4a8, cuda, K, S, dtype, post):
    g = torch.Generator(device="cuda").manual_seed(K)
    h = torch.randn(S, K, generator=g, device=cuda).to(torch.bfloat16 if dtype == "bf16" else torch.float32)
    zero = torch.zeros_like(h)
    many, one = torch.empty_like(h), torch.empty_like(h[:1])
    for i in range(150):
        ss = float((h[i].double() ** 2).sum())
        eps = border(ss, K, 1.3 + 0.01 * (i % 40))
        if post:                                              # the norm of what is added
            n = w4a8.Norm.of(K, variant=-1, eps=eps, post_variant=2, dtype=dtype)
            w4a8.launch_add_norm(n, zero, h, S, H_out=many)
            w4a8.launch_add_norm(n, zero, h[i:], 1, H_out=one)
        else:
            n = w4a8.Norm.of(K, variant=2, eps=eps, dtype=dtype)
            w4a8.launch_add_norm(n, h, None, S, N=many)
            w4a8.launch_add_norm(n, h[i:], None, 1, N=one)
        a, b = one[0].double(), many[i].double()
        # r one step apart, 2^-23; the product with it rounded on either side, 2^-24 each (a sum with zero is exact); bf16 outputs rounded once more, 2^-8 each
        assert ((a - b).abs() <= (2.0 ** -22 + (2.0 ** -7 if dtype == "bf16" else 0.0)) * a.abs()).all(), i
        # away from the border, with the same sums, the bits are the same
        n.eps = eps * (1 + 1e-5)
        w4a8.launch_add_norm(n, zero if post else h, h if post else None, S, **{"H_out" if post else "N": many})
        w4a8.launch_add_norm(n, zero[i:] if post else h[i:], h[i:] if post else None, 1, **{"H_out" if post else "N": one})
        assert torch.equal(one[0], many[i]), i
