"""Norms of heads whose squares fp32 does not hold (w4a8_rope_qk): elements around 2e18 and above, and tiny ones without an eps."""
import pytest
import torch

from layer_plain import DTYPES, U, near, norm
from test_gpu_rope import _turn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("size,eps", [(2e18, 1e-6), (1e19, 1e-6), (3e25, 0.0), (1e37, 1e-6), (1e-18, 0.0), (1e-22, 0.0), (1e-30, 0.0), (1e-37, 0.0), (1e-20, 1e-44), (1.0, 0.0)])
@pytest.mark.parametrize("D,R,variant", [(128, 128, 0), (128, 64, 2), (80, 40, 1), (256, 0, 0)])
def test_norms_of_huge_and_tiny_heads(w4a8, cuda, D, R, variant, size, eps, dtype):
    Hq, Hkv = 5, 2
    for T in (3, 700):
        g = torch.Generator(device="cuda").manual_seed(T + D)
        rows = torch.randn(T, (Hq + Hkv) * D, generator=g, device=cuda)
        rows[:, : 3 * D] *= size                              # some heads only: those beside them are ordinary
        rows = rows.to(DTYPES[dtype])
        position = torch.randint(0, 1000, (T,), generator=g, device=cuda, dtype=torch.int32)
        w = [torch.rand(D, generator=g, device=cuda) + 0.5 if variant in (0, 1) else None for _ in range(2)]
        rope = w4a8.Rope.of(D, R, 10000.0, "none", False, w[0], w[1], variant, eps, device=cuda)
        q, k = torch.empty(T, Hq * D, dtype=rows.dtype, device=cuda), torch.empty(T, Hkv * D, dtype=rows.dtype, device=cuda)
        cols = (Hq + Hkv) * D
        w4a8.launch_rope_qk(rope, rows, cols, Hq, rows[:, Hq * D:], cols, Hkv, position, T, q, Hq * D, k, Hkv * D, dtype)
        for out, lo, H, wt in ((q, 0, Hq, w[0]), (k, Hq, Hkv, w[1])):
            x = norm(rows[:, lo * D:(lo + H) * D].double().reshape(T * H, D), wt, variant, eps).view(T, H, D)
            want, bound = _turn(x, position, R, 10000.0, False)
            near(out, want.reshape(T, -1), (20 * U * bound + bound * position.double()[:, None, None] * 2.0 ** -50).reshape(T, -1), "turned")
        w4a8.launch_rope_qk(rope, rows, cols, Hq, rows[:, Hq * D:], cols, Hkv, position, T, dtype=dtype)           # in place: the same bits
        assert torch.equal(rows[:, : Hq * D], q) and torch.equal(rows[:, Hq * D:], k)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_numbers_that_are_none_stay_in_their_head(w4a8, cuda, dtype):
    T, H, D = 40, 9, 64
    rows = torch.randn(T, H * D, device=cuda).to(DTYPES[dtype])
    position = torch.arange(T, dtype=torch.int32, device=cuda)
    rope, clean = w4a8.Rope.of(D, D, variant=2, device=cuda), rows.clone()
    w4a8.launch_rope_qk(rope, clean, H * D, H, None, 0, 0, position, T, dtype=dtype)
    rows[::3, 2 * D + 5], rows[1::3, 4 * D + 7] = float("nan"), float("inf")
    w4a8.launch_rope_qk(rope, rows, H * D, H, None, 0, 0, position, T, dtype=dtype)
    touched = torch.zeros(T, H, dtype=torch.bool, device=cuda)
    touched[::3, 2], touched[1::3, 4] = True, True
    got, want = rows.view(T, H, D), clean.view(T, H, D)
    assert torch.equal(got[~touched], want[~touched]) and torch.isnan(got[::3, 2]).all() and torch.isnan(got[1::3, 4, 7]).all()
