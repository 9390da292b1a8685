"""Residual add and norms (w4a8_add_norm) against the formula in 64 bits, its codes against the definition's fp32 steps bit for bit."""
import pytest
import torch

from layer_plain import DTYPES, U, add_norm, add_norm32, near, quantize

pytestmark = pytest.mark.gpu
EPS = 1e-6


def _inputs(S, K, dtype, y_dtype, variant, post, gate, seed, ld=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")
    rows = lambda dt: torch.cat((r(S, K) * torch.exp(0.5 * r(S, 1)), r(S, ld)), 1).to(DTYPES[dt])
    w = r(K) * 0.2 + 1 if variant in (0, 1) else None
    pw = r(K) * 0.2 + 1 if post in (0, 1) else None
    gt = {"": None, "channel": r(K), "token": r(S, K)}[gate]
    return rows(dtype), rows(y_dtype), w, pw, gt


def _slack(p, s, n, h):
    """p carries at most six roundings (the factor, two products or the sum 1 + w among them, gate, alpha), h' one more; n's factor follows h' in the mean and is
    rounded, then two products and a sum."""
    of_s = U * (6 * p.abs() + s.abs())
    if n is s:
        return of_s, of_s
    rms = lambda v: (v * v).mean(1, keepdim=True).sqrt()
    carried = of_s * (n.abs() / s.abs().clamp(min=1e-300))
    mean = 6 * rms(p) / rms(s).clamp(min=1e-30) + 1
    return of_s, carried + U * n.abs() * (mean + 5)


CASES = [(1, 32), (3, 64), (5, 96), (2, 256), (149, 288), (1, 5120), (7, 3840), (200, 1024), (150, 8192), (1, 8192), (1, 8224), (2, 16384), (160, 16384), (2, 16416), (3, 32768)]


@pytest.mark.parametrize("dtype,y_dtype", [("fp32", "fp32"), ("bf16", "bf16"), ("bf16", "fp32"), ("fp16", "fp16"), ("fp16", "fp32")])
@pytest.mark.parametrize("S,K", CASES)
def test_sum_and_norm_follow_the_formula(w4a8, cuda, S, K, dtype, y_dtype):
    i = CASES.index((S, K))
    for variant, post, gate, alpha in [((0, 1, 2)[i % 3], -1, "", 1.0), (0, (0, 1, 2)[i % 3], ("channel", "token")[i % 2], 0.22), (-1, 0, "token", -1.5)]:
        h, y, w, pw, gt = _inputs(S, K, dtype, y_dtype, variant, post, gate, 10 * i + variant)
        norm = w4a8.Norm.of(K, w, variant, EPS, pw, post, gt, alpha, dtype, y_dtype)
        ho, n = torch.empty_like(h), torch.empty_like(h)
        w4a8.launch_add_norm(norm, h, y, S, H_out=ho, N=n)
        p, s, want = add_norm(h, y, w, variant, pw, post, gt, alpha, EPS)
        of_s, of_n = _slack(p, s, s if variant == -1 else want, h)
        near(ho, s, of_s, "h'")
        near(n, want, of_n, "n")


@pytest.mark.parametrize("dtype,y_dtype", [("fp32", "fp32"), ("bf16", "fp32"), ("fp16", "fp16")])
@pytest.mark.parametrize("S,K", [(1, 32), (1, 5120), (5, 96), (150, 3840), (2, 8224), (3, 32768), (300, 160)])
@pytest.mark.parametrize("group", [32, 0])
def test_codes_are_those_of_the_definition(w4a8, cuda, S, K, dtype, y_dtype, group):
    h, y, w, pw, gt = _inputs(S, K, dtype, y_dtype, 0, 1, "channel", 77 + K)
    h[S // 2] = 0
    y[S // 2] = 0                                                     # a row of zeros: scale 0, codes 0
    norm = w4a8.Norm.of(K, w, 0, EPS, pw, 1, gt, 0.7, dtype, y_dtype)
    nb = 1 if group == 0 else K // 32
    xq = torch.full((S + 1, K), 99, dtype=torch.int8, device=cuda)
    xs = torch.full((S + 1, nb), 7.0, device=cuda)
    xsum = torch.full((S + 1, nb), 5, dtype=torch.int32, device=cuda)
    n = torch.empty_like(h)
    w4a8.launch_add_norm(norm, h, y, S, N=n, xq=xq, xs=xs, xsum=None if group == 0 else xsum, group=group)
    _, n32 = add_norm32(h, y, w, 0, pw, 1, gt, 0.7, EPS)
    q, scale, total = quantize(n32, group)
    assert torch.equal(n, n32.to(n.dtype))
    assert torch.equal(xq[:S], q) and torch.equal(xs[:S], scale) and (group == 0 or torch.equal(xsum[:S], total))
    assert (xq[S] == 99).all() and (xs[S] == 7).all() and (xsum[S] == 5).all()       # behind the last row
    if group == 32 and dtype == "fp32":                                # the quantizer on its own gives the same
        q2, s2, t2 = torch.empty_like(q), torch.empty_like(scale), torch.empty_like(total)
        w4a8.launch_quantize_x_q8(n, q2, s2, t2, K, S)
        assert torch.equal(q2, q) and torch.equal(s2, scale) and torch.equal(t2, total)


def test_bits_of_a_row_do_not_depend_on_the_others(w4a8, cuda):
    K = 5120
    h, y, w, pw, _ = _inputs(400, K, "fp32", "fp32", 0, 0, "", 5)
    norm = w4a8.Norm.of(K, w, 0, EPS, pw, 0)
    one, many = (torch.empty_like(h) for _ in range(2))
    w4a8.launch_add_norm(norm, h, y, 400, N=many)                      # wide rows of threads for a few rows, narrow ones for many
    for r in (0, 123, 399):
        w4a8.launch_add_norm(norm, h[r:], y[r:], 1, N=one)
        assert torch.equal(one[0], many[r])


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_pitches_and_in_place(w4a8, cuda, dtype):
    S, K, pad = 37, 416, 24
    h, y, w, _, _ = _inputs(S, K, dtype, dtype, 1, -1, "", 9, ld=pad)
    norm = w4a8.Norm.of(K, w, 1, EPS, dtype=dtype)
    ho, n = torch.full_like(h, 3), torch.full_like(h, 4)
    w4a8.launch_add_norm(norm, h, y, S, H_out=ho, N=n, ldh=K + pad, ldy=K + pad, ldo=K + pad, ldn=K + pad)
    assert (ho[:, K:] == 3).all() and (n[:, K:] == 4).all()
    h2, y2 = h.clone(), y.clone()
    w4a8.launch_add_norm(norm, h2, y2, S, H_out=h2, N=y2, ldh=K + pad, ldy=K + pad, ldo=K + pad, ldn=K + pad)     # the stream's memory and the block's output's
    assert torch.equal(h2[:, :K], ho[:, :K]) and torch.equal(y2[:, :K], n[:, :K])
    assert torch.equal(h2[:, K:], h[:, K:]) and torch.equal(y2[:, K:], y[:, K:])
    side = torch.zeros(S, 2 * K, dtype=h.dtype, device=cuda)           # columns of one buffer side by side
    side[:, :K] = h[:, :K]
    w4a8.launch_add_norm(norm, side, y, S, N=side[:, K:], ldh=2 * K, ldy=K + pad, ldn=2 * K)
    assert torch.equal(side[:, K:], n[:, :K]) and torch.equal(side[:, :K], h[:, :K])


def test_without_a_block_output_it_is_the_norm(w4a8, cuda):
    h, _, w, _, _ = _inputs(9, 640, "fp16", "fp16", 0, -1, "", 3)
    n, ho = torch.empty_like(h), torch.empty_like(h)
    w4a8.launch_add_norm(w4a8.Norm.of(640, w, 0, EPS, dtype="fp16"), h, None, 9, H_out=ho, N=n)
    _, s, want = add_norm(h, None, w, 0, None, -1, None, 1.0, EPS)
    assert torch.equal(ho, h)
    near(n, want, 8 * U * want.abs(), "n")


def test_numbers_that_are_none_stay_in_their_row(w4a8, cuda):
    h, y, w, _, _ = _inputs(5, 320, "fp32", "fp32", 0, -1, "", 4)
    y[1, 7], y[3, 9] = float("nan"), float("inf")
    n = torch.empty_like(h)
    w4a8.launch_add_norm(w4a8.Norm.of(320, w, 0, EPS), h, y, 5, N=n)
    _, _, want = add_norm(h, y, w, 0, None, -1, None, 1.0, EPS)
    ok = torch.tensor([0, 2, 4], device=cuda)
    near(n[ok], want[ok], 1e-5 * want[ok].abs() + 1e-5, "n")
    assert torch.isnan(n[1]).all() and torch.isnan(n[3, 9]) and (n[3, :9] == 0).all()


def test_captured_replayed_and_on_another_stream(w4a8, cuda):
    S, K = 33, 2048
    h, y, w, _, _ = _inputs(S, K, "fp32", "fp32", 0, -1, "", 6)
    norm, n = w4a8.Norm.of(K, w, 0, EPS), torch.empty_like(h)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        w4a8.launch_add_norm(norm, h, y, S, N=n)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            w4a8.launch_add_norm(norm, h, y, S, H_out=h, N=n)
            w4a8.launch_add_norm(norm, h, y, S, H_out=h, N=n)
        want_h = h + y + y
        graph.replay()
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    assert torch.equal(h, want_h) and torch.equal(n, add_norm32(h, None, w, 0, None, -1, None, 1.0, EPS)[1])
