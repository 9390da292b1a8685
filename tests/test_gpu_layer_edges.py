"""Calls of the layer operators that the documentation allows and the other tests do not make: the smallest and largest sizes, several calls at once,
structs without tensors, rows of odd pitch."""
import numpy as np
import pytest
import torch

from layer_plain import DTYPES, U, add_norm, add_norm32, near, norm, quantize
from test_gpu_moe_route import check
from test_gpu_moe_route import plain as plain_route
from test_gpu_rope import _turn

pytestmark = pytest.mark.gpu


def test_a_gate_for_each_token_of_a_wider_buffer(w4a8, cuda):
    S, K = 21, 480
    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.randn(s, generator=g, device=cuda)
    h, y, wide = r(S, K), r(S, K), r(S, 3 * K)
    gate = wide[:, K:2 * K]
    n = w4a8.Norm.of(K, variant=2, gate=gate, alpha=0.3)
    out = torch.empty_like(h)
    w4a8.launch_add_norm(n, h, y, S, N=out)
    assert torch.equal(out, add_norm32(h, y, None, 2, None, -1, gate, 0.3, 1e-6)[1])
    with pytest.raises(ValueError, match="a gate of 21"):
        w4a8.launch_add_norm(n, torch.cat((h, h)), torch.cat((y, y)), 2 * S, N=torch.cat((out, out)))
    one = w4a8.Norm.of(K, variant=2, gate=gate[:1].clone(), alpha=0.3)             # one row: the channels' gate for all
    w4a8.launch_add_norm(one, h, y, S, N=out)
    assert torch.equal(out, add_norm32(h, y, None, 2, None, -1, gate[0], 0.3, 1e-6)[1])


def test_every_output_of_a_norm_at_once_and_alone(w4a8, cuda):
    """n in its own type, codes of blocks and codes of rows do not change with what else is asked for."""
    S, K = 5, 1056
    h, y = torch.randn(S, K, device=cuda).bfloat16(), torch.randn(S, K, device=cuda)
    w = torch.rand(K, device=cuda) + 0.5
    n = w4a8.Norm.of(K, w, 1, dtype="bf16", y_dtype="fp32")
    want_s, want_n = add_norm32(h, y, w, 1, None, -1, None, 1.0, 1e-6)
    for group in (32, 0):
        q, scale, total = quantize(want_n, group)
        for both in (True, False):
            xq, xs, xsum = torch.empty_like(q), torch.empty_like(scale), torch.empty_like(total)
            out, s = torch.empty_like(h), torch.empty_like(h)
            w4a8.launch_add_norm(n, h, y, S, H_out=s if both else None, N=out if both else None, xq=xq, xs=xs, xsum=xsum if group and both else None, group=group)
            assert torch.equal(xq, q) and torch.equal(xs, scale)
            if both:
                assert torch.equal(s, want_s.bfloat16()) and torch.equal(out, want_n.bfloat16()) and (not group or torch.equal(xsum, total))


def test_rows_too_long_for_one_pass_of_loads(w4a8, cuda):
    """Rows between the quantizer's kernels: 8192, 16384 and 32768 elements and a block more or less, few rows and many."""
    for K in (8160, 8192, 8224, 16352, 16384, 16416, 32736, 32768):
        for S in (1, 2, 150):
            x = torch.randn(S, K, device=cuda)
            xq, xs = torch.empty(S, K, dtype=torch.int8, device=cuda), torch.empty(S, device=cuda)
            w4a8.launch_quantize_rows_q8(x, K, S, K, xq, xs)
            q, scale, _ = quantize(x, 0)
            assert torch.equal(xq, q) and torch.equal(xs, scale[:, 0]), (K, S)


def test_scales_at_the_ends_of_fp32(w4a8, cuda):
    """Rows of subnormal, tiny and huge elements, and of infinities: codes and scales of the definition, products of them what fp32 makes."""
    K, N = 64, 40
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(8, K, generator=g, device=cuda)
    x[0] *= 1e-42
    x[1] *= 1e-37
    x[2] *= 1e37
    x[3] *= 2.0 ** -100
    x[4, 5] = float("inf")
    x[5, 6] = float("nan")
    x[6] = 0
    xq, xs = torch.empty(8, K, dtype=torch.int8, device=cuda), torch.empty(8, device=cuda)
    w4a8.launch_quantize_rows_q8(x, K, 8, K, xq, xs)
    for r in (0, 1, 2, 3, 6, 7):
        q, scale, _ = quantize(x[r:r + 1], 0)
        assert torch.equal(xq[r:r + 1], q) and torch.equal(xs[r:r + 1], scale[:, 0]), r
    assert torch.isinf(xs[4]) and (xq[4] == 0).all() and torch.isfinite(xs[5]) and xq[5, 6] == 0
    wq, ws = torch.randint(-127, 128, (N, K), generator=g, device=cuda, dtype=torch.int8), torch.rand(N, generator=g, device=cuda)
    Y = torch.empty(8, N, device=cuda)
    w4a8.launch_gemm_w8a8(xq, xs, wq, ws, Y, N, 8, N, K)
    want = (xq.double() @ wq.double().T).float() * xs[:, None] * ws
    ok = torch.tensor([0, 1, 2, 3, 6, 7], device=cuda)
    assert torch.equal(Y[ok], want[ok]) and torch.isnan(Y[4]).all()                # 0 * inf


@pytest.mark.parametrize("heads_q,heads_k", [(0, 3), (5, 0), (1, 1), (131, 70)])
def test_queries_or_keys_alone(w4a8, cuda, heads_q, heads_k):
    D, T = 16, 7
    rope = w4a8.Rope.of(D, 8, interleaved=True, device=cuda)
    position = torch.tensor([0, 1, 5, -1, 100000, 2 ** 31 - 1, 3], dtype=torch.int32, device=cuda)
    q, k = (torch.randn(T, max(1, h) * D, device=cuda) for h in (heads_q, heads_k))
    qo, ko = q.clone(), k.clone()
    w4a8.launch_rope_qk(rope, qo if heads_q else None, max(1, heads_q) * D, heads_q, ko if heads_k else None, max(1, heads_k) * D, heads_k, position, T)
    for x, out, h in ((q, qo, heads_q), (k, ko, heads_k)):
        if not h:
            assert torch.equal(x, out)
            continue
        want, size = _turn(x.double().view(T, h, D), position.clamp(min=0), 8, 10000.0, True)
        there = (position >= 0) & (position < 2 ** 30)
        near(out[there], want.reshape(T, -1)[there], (size * (20 * U + position.clamp(min=0).double()[:, None, None] * 2.0 ** -50)).reshape(T, -1)[there], "turned")
        assert torch.equal(out[3], x[3]) and torch.isfinite(out).all()


def test_several_calls_at_once(w4a8, cuda):
    """All operators side by side on four streams, over and over: no call sees another one's data."""
    S, K, N, E = 64, 1024, 768, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s: torch.randn(s, generator=g, device=cuda)
    w = r(K) * 0.1 + 1
    nrm, router = w4a8.Norm.of(K, w), w4a8.Router.of(E, 4)
    rope = w4a8.Rope.of(64, 64, device=cuda)
    wq, ws = torch.randint(-127, 128, (N, K), generator=g, device=cuda, dtype=torch.int8), torch.rand(N, generator=g, device=cuda)
    position = torch.arange(S, dtype=torch.int32, device=cuda) * 31
    jobs = []
    for i in range(4):
        jobs.append({"h": r(S, K), "y": r(S, K), "logits": r(S, E), "n": torch.empty(S, K, device=cuda), "q": torch.empty(S, K, device=cuda), "xq": torch.empty(S, K, dtype=torch.int8, device=cuda),
                     "xs": torch.empty(S, device=cuda), "Y": torch.empty(S, N, device=cuda), "idx": torch.empty(S, 4, dtype=torch.int32, device=cuda), "weight": torch.empty(S, 4, device=cuda)})
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(10):
        for st, j in zip(streams, jobs):
            with torch.cuda.stream(st):
                w4a8.launch_add_norm(nrm, j["h"], j["y"], S, N=j["n"])
                w4a8.launch_rope_qk(rope, j["n"], K, 16, None, 0, 0, position, S, j["q"], K)
                w4a8.linear_w8a8(j["n"], K, j["xq"], j["xs"], wq, ws, j["Y"], N, S, N, K)
                w4a8.launch_moe_route(router, j["logits"], E, S, j["idx"], j["weight"])
    torch.cuda.synchronize()
    for j in jobs:
        _, n = add_norm32(j["h"], j["y"], w, 0, None, -1, None, 1.0, 1e-6)
        q, scale, _ = quantize(n, 0)
        assert torch.equal(j["n"], n) and torch.equal(j["Y"], (q.double() @ wq.double().T).float() * scale * ws)
        want, size = _turn(n.double().view(S, 16, 64), position, 64, 10000.0, False)
        near(j["q"], want.view(S, K), (size * (20 * U + position.double()[:, None, None] * 2.0 ** -50)).view(S, K), "turned")
        assert np.array_equal(j["idx"].cpu().numpy(), plain_route(j["logits"], 4)[0])
    w4a8.device_status()


def test_near_choices_of_many_tokens(w4a8, cuda):
    """Logits so close that fp32 scores cannot tell them apart: the choices of fp64, by candidates or over the whole token."""
    g = torch.Generator(device="cuda").manual_seed(4)
    for E, spread in ((64, 1e-5), (256, 1e-6), (512, 1e-6), (40, 1e-7)):
        logits = 1.0 + spread * torch.randn(200, E, generator=g, device=cuda)
        bias = 1e-6 * torch.randn(E, generator=g, device=cuda)
        for how in (dict(scoring="sigmoid"), dict(scoring="sigmoid", bias=bias), dict(scoring="softmax", bias=bias), dict(scoring="sigmoid", bias=bias, groups=8, topk_groups=3, group_score="sum2"),
                    dict(scoring="softmax", groups=4, topk_groups=2, group_score="sum2")):
            check(w4a8, logits, 6, **how)
    mixed = torch.randn(300, 128, generator=g, device=cuda)
    mixed[:, 64:68] = mixed.amax(1, keepdim=True) * (1 + 1e-7 * torch.randn(300, 4, generator=g, device=cuda))    # a few near values among many
    for how in (dict(scoring="sigmoid"), dict(scoring="softmax", bias=torch.zeros(128, device=cuda)), dict(scoring="sigmoid", groups=2, topk_groups=1)):
        check(w4a8, mixed, 8, **how)


def test_the_largest_products_of_a_serving_step(w4a8, cuda):
    """A vocabulary's outputs for one row and for a few, past 2^31 bytes of weights' reach of a tile, against sums of a sample of channels."""
    M, N, K = 3, 151936, 4096
    g = torch.Generator(device="cuda").manual_seed(5)
    xq = torch.randint(-127, 128, (M, K), generator=g, device=cuda, dtype=torch.int8)
    wq = torch.randint(-127, 128, (N, K), generator=g, device=cuda, dtype=torch.int8)
    xs, ws = torch.rand(M, generator=g, device=cuda), torch.rand(N, generator=g, device=cuda) * 1e-4
    Y = torch.empty(M, N, device=cuda)
    w4a8.launch_gemm_w8a8(xq, xs, wq, ws, Y, N, M, N, K)
    at = torch.cat((torch.arange(0, N, 997, device=cuda), torch.arange(N - 300, N, device=cuda)))
    want = (xq.double() @ wq[at].double().T).float() * xs[:, None] * ws[at]
    assert torch.equal(Y[:, at], want)
    w4a8.device_status()


@pytest.mark.parametrize("dtype,y_dtype", [("fp32", "fp32"), ("bf16", "fp32"), ("fp16", "fp16")])
@pytest.mark.parametrize("S,K", [(593, 32), (601, 96), (1203, 256), (602, 512), (700, 544), (605, 1024)])
def test_short_rows_in_great_number(w4a8, cuda, S, K, dtype, y_dtype):
    """Rows that a warp has to itself: the definition's bits in every output, nothing behind the last row, and the same bits as a row by itself."""
    g = torch.Generator(device="cuda").manual_seed(K)
    r = lambda *s: torch.randn(s, generator=g, device=cuda)
    h, y, w, pw = r(S + 1, K).to(DTYPES[dtype]), r(S + 1, K).to(DTYPES[y_dtype]), r(K) * 0.1 + 1, r(K) * 0.1
    for yy, post, group in ((y, 1, 32), (y, -1, 0), (None, -1, 0), (None, -1, 32)):
        n = w4a8.Norm.of(K, w, 0, 1e-6, pw, post, None, 0.7, dtype, y_dtype)
        blocks = 1 if group == 0 else K // 32
        s_out, out = (torch.full((S + 1, K), 3.0, device=cuda).to(h.dtype) for _ in range(2))
        xq, xs = torch.full((S + 1, K), 99, dtype=torch.int8, device=cuda), torch.full((S + 1, blocks), 7.0, device=cuda)
        w4a8.launch_add_norm(n, h, yy, S, H_out=s_out, N=out, xq=xq, xs=xs, group=group)
        want_s, want = add_norm32(h, yy, w, 0, pw, post, None, 0.7, 1e-6)
        q, scale, _ = quantize(want, group)
        assert torch.equal(s_out[:S], want_s[:S].to(h.dtype)) and torch.equal(out[:S], want[:S].to(h.dtype))
        assert torch.equal(xq[:S], q[:S]) and torch.equal(xs[:S], scale[:S])
        assert (s_out[S] == 3).all() and (out[S] == 3).all() and (xq[S] == 99).all() and (xs[S] == 7).all()
        one = torch.empty(1, K, device=cuda).to(h.dtype)
        w4a8.launch_add_norm(n, h[17:], None if yy is None else yy[17:], 1, N=one)
        assert torch.equal(one[0], out[17])
    xq, xs = torch.empty(S, K, dtype=torch.int8, device=cuda), torch.empty(S, device=cuda)
    w4a8.launch_quantize_rows_q8(h, K, S, K, xq, xs, dtype)
    q, scale, _ = quantize(h[:S].float(), 0)
    assert torch.equal(xq, q) and torch.equal(xs, scale[:, 0])
