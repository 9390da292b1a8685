"""Norms and rotary positions of queries and keys (w4a8_rope_qk) against complex products in 64 bits."""
import math

import pytest
import torch

from layer_plain import DTYPES, U, near, norm

pytestmark = pytest.mark.gpu
EPS = 1e-6


def _turn(x, position, R, base, interleaved, magnitude=1.0, factor=1.0):
    """x[T][H][D] in 64 bits -> its first R elements turned, and |a| + |b| of each element's pair."""
    T, H, D = x.shape
    f = torch.tensor([base ** (-2.0 * i / R) / factor for i in range(R // 2)], dtype=torch.float64, device=x.device)
    # modulo a turn in whole numbers where a double would lose the fraction: positions go up to 2^31
    turns = torch.tensor([(base ** (-2.0 * i / R) / factor) / (2 * math.pi) for i in range(R // 2)], dtype=torch.float64, device=x.device)
    a = position.double()[:, None] * turns
    angle = (a - a.floor()) * (2 * math.pi)
    z = torch.polar(torch.full_like(angle, magnitude), angle)[:, None]
    out, size = x.clone(), x.abs()
    if R:
        p, q = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
        t = torch.complex(x[..., p].contiguous(), x[..., q].contiguous()) * z
        out[..., p], out[..., q] = t.real, t.imag
        s = (x[..., p].abs() + x[..., q].abs()) * magnitude
        size[..., p], size[..., q] = s, s
    del f
    return out, size


CASES = [
    # T, Hq, Hkv, D, rotary, interleaved, variant, far
    (1, 32, 8, 128, 128, 0, 0, 413), (64, 32, 8, 128, 128, 0, -1, 131072), (7, 4, 4, 64, 64, 1, -1, 1000), (5, 3, 1, 80, 32, 0, 1, 5000),
    (33, 7, 1, 96, 24, 1, 2, 99999), (9, 2, 2, 256, 256, 0, 0, 2 ** 20), (3, 5, 1, 256, 8, 1, 0, 77), (600, 16, 2, 128, 64, 0, 0, 40000), (300, 28, 4, 128, 128, 1, 2, 10),
    (4, 1, 1, 8, 8, 0, 0, 50), (2, 40, 8, 112, 0, 0, 0, 50), (1500, 9, 3, 64, 40, 0, -1, 3000), (11, 64, 1, 16, 16, 1, 1, 4),
]


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("case", CASES)
def test_norms_and_rotations_follow_the_formula(w4a8, cuda, case, dtype):
    T, Hq, Hkv, D, R, inter, variant, far = case
    g = torch.Generator(device="cuda").manual_seed(T + D + R)
    cols = (Hq + 2 * Hkv) * D
    rows = torch.randn(T, cols, generator=g, device=cuda).to(DTYPES[dtype])
    position = torch.randint(0, far, (T,), generator=g, device=cuda, dtype=torch.int32)
    if T > 2:
        position[1] = -1
    w = [torch.randn(D, generator=g, device=cuda) * 0.2 + 1 if variant in (0, 1) else None for _ in range(2)]
    rope = w4a8.Rope.of(D, R, 10000.0, "none", bool(inter), w[0], w[1], variant, EPS, device=cuda)
    q_out, k_out = (torch.full((T + 1, H * D + 8), 5.0, device=cuda).to(rows.dtype) for H in (Hq, Hkv))
    before = rows.clone()
    w4a8.launch_rope_qk(rope, rows, cols, Hq, rows[:, Hq * D:], cols, Hkv, position, T, q_out, Hq * D + 8, k_out, Hkv * D + 8, dtype)
    assert torch.equal(rows, before)
    there = position >= 0
    for out, lo, H, wt in ((q_out, 0, Hq, w[0]), (k_out, Hq, Hkv, w[1])):
        x = rows[:, lo * D:(lo + H) * D].double().reshape(T * H, D)
        want, size = _turn(norm(x, wt, variant, EPS).view(T, H, D), position.clamp(min=0), R, 10000.0, inter)
        # angle 2^-25 half turns and the frequency's own 2^-52 * position, cosine and sine 2 ulp, their products and sum 3, norm 12
        slack = size * (20 * U + 2 * math.pi * position.clamp(min=0).double()[:, None, None] * 2.0 ** -53)
        near(out[:T, :H * D][there], want.reshape(T, H * D)[there], slack.reshape(T, H * D)[there], "turned")
        assert (out[:T, :H * D][~there] == 5).all() and (out[T] == 5).all() and (out[:, H * D:] == 5).all()
    # in place: the same bits, values and rows without a request as they were
    w4a8.launch_rope_qk(rope, rows, cols, Hq, rows[:, Hq * D:], cols, Hkv, position, T, dtype=dtype)
    assert torch.equal(rows[there][:, : Hq * D], q_out[:T, :Hq * D][there]) and torch.equal(rows[there][:, Hq * D:(Hq + Hkv) * D], k_out[:T, :Hkv * D][there])
    assert torch.equal(rows[:, (Hq + Hkv) * D:], before[:, (Hq + Hkv) * D:]) and torch.equal(rows[~there], before[~there])


def test_far_positions_lose_nothing(w4a8, cuda):
    """A frequency of 1 / 32 turn has whole numbers of turns that are exact in binary: positions near 2^31 turn as small ones do."""
    D, turns = 64, torch.full((32,), 1 << 59, dtype=torch.int64, device=cuda)
    rope = w4a8.Rope.of(D, D, device=cuda)
    rope.turns = turns.data_ptr()
    x = torch.randn(2, D, device=cuda)
    for far in (2 ** 31 - 1, 2 ** 31 - 32, 2 ** 30 + 5):
        rows = torch.stack((x[0], x[0]))
        position = torch.tensor([far, far % 32], dtype=torch.int32, device=cuda)
        w4a8.launch_rope_qk(rope, rows, D, 1, None, 0, 0, position, 2)
        assert torch.equal(rows[0], rows[1])
        a = 2 * math.pi * (far % 32) / 32
        want = torch.cat((x[0, :32] * math.cos(a) - x[0, 32:] * math.sin(a), x[0, 32:] * math.cos(a) + x[0, :32] * math.sin(a))).double()
        near(rows[0], want, 30 * U * (x[0, :32].abs() + x[0, 32:].abs()).repeat(2).double(), "turned")


def test_magnitude_and_scaled_frequencies(w4a8, cuda):
    D, T = 128, 50
    x = torch.randn(T, D, device=cuda)
    position = torch.arange(T, dtype=torch.int32, device=cuda) * 700
    rope = w4a8.Rope.of(D, 96, 10000.0, "linear", factor=4.0, magnitude=1.25, device=cuda)
    got = x.clone()
    w4a8.launch_rope_qk(rope, got, D, 1, None, 0, 0, position, T)
    want, size = _turn(x.double().view(T, 1, D), position, 96, 10000.0, False, 1.25, 4.0)
    near(got, want.view(T, D), (20 * U * size + size * position.double()[:, None, None] * 2.0 ** -50).view(T, D), "turned")


def test_captured_and_replayed(w4a8, cuda):
    T, D = 16, 128
    rows = torch.randn(T, 10 * D, device=cuda)
    position = torch.arange(T, dtype=torch.int32, device=cuda)
    rope = w4a8.Rope.of(D, D, device=cuda)
    q, k = torch.empty(T, 8 * D, device=cuda), torch.empty(T, D, device=cuda)
    call = lambda: w4a8.launch_rope_qk(rope, rows, 10 * D, 8, rows[:, 8 * D:], 10 * D, 1, position, T, q, 8 * D, k, D)
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    position += 1000
    rows += 1
    graph.replay()
    a, b = q.clone(), k.clone()
    call()
    torch.cuda.synchronize()
    assert torch.equal(a, q) and torch.equal(b, k)
