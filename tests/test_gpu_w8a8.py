"""8-bit products with scales for each row and channel: the sums are exact, so outputs are compared bit for bit with the definition's fp32 steps."""
import pytest
import torch

from layer_plain import DTYPES, quantize

pytestmark = pytest.mark.gpu


def _case(M, N, K, seed, bias=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    xq = torch.randint(-127, 128, (M, K), generator=g, device="cuda", dtype=torch.int8)
    wq = torch.randint(-128, 128, (N, K), generator=g, device="cuda", dtype=torch.int8)
    xs, ws = torch.rand(M, generator=g, device="cuda") * 0.1, torch.rand(N, generator=g, device="cuda") * 1e-3
    return xq, xs, wq, ws, torch.randn(N, generator=g, device="cuda") if bias else None


def _want(xq, xs, wq, ws, b, dtype):
    y = (xq.double() @ wq.double().T).float() * xs[:, None] * ws           # whole numbers below 2^53: the double is exact, rounded once
    return (y if b is None else y + b).to(DTYPES[dtype])


def _run(w4a8, case, dtype, ld=0):
    xq, xs, wq, ws, b = case
    M, N, K = xq.shape[0], wq.shape[0], xq.shape[1]
    Y = torch.full((M + 1, N + ld), 3.0, device=xq.device).to(DTYPES[dtype])
    w4a8.launch_gemm_w8a8(xq, xs, wq, ws, Y, N + ld, M, N, K, dtype, bias=b)
    assert (Y[M] == 3).all() and (Y[:, N:] == 3).all()
    return Y[:M, :N]


@pytest.mark.parametrize("K", [32, 96, 128, 416, 2048])
@pytest.mark.parametrize("M,N", [(1, 1), (1, 128), (2, 300), (7, 5), (16, 129), (17, 1000), (33, 64), (64, 640), (65, 127), (100, 4091), (128, 256), (129, 700), (256, 130), (257, 1), (300, 999), (777, 257)])
def test_products_are_exact(w4a8, cuda, M, N, K):
    case = _case(M, N, K, M + N + K, bias=(M + N) % 2 == 0)
    for dtype, ld in (("fp32", 0), ("bf16", 1), ("fp16", 5)):
        assert torch.equal(_run(w4a8, case, dtype, ld), _want(*case, dtype)), dtype
    w4a8.device_status()


@pytest.mark.parametrize("M,N,K", [(1, 17408, 5120), (16, 3840, 15360), (5, 128, 32768), (40, 512, 16416), (2048, 1024, 512), (333, 4091, 3840), (8, 60000, 256), (1000, 3000, 1056), (64, 6144, 5120)])
def test_larger_products(w4a8, cuda, M, N, K):
    case = _case(M, N, K, K, bias=False)
    assert torch.equal(_run(w4a8, case, "fp32"), _want(*case, "fp32"))
    w4a8.device_status()


def test_the_largest_sums_fit(w4a8, cuda):
    K = 131040
    xq, wq = torch.full((3, K), -128, dtype=torch.int8, device=cuda), torch.full((5, K), -128, dtype=torch.int8, device=cuda)
    xq[1], wq[2] = 127, 127
    one = torch.ones(5, device=cuda)
    case = (xq, one[:3].clone(), wq, one, None)
    assert torch.equal(_run(w4a8, case, "fp32"), _want(*case, "fp32"))


def test_bits_do_not_depend_on_the_rows_of_a_call(w4a8, cuda):
    case = _case(300, 520, 1312, 3)
    whole = _run(w4a8, case, "fp32").clone()
    for lo, n in ((0, 1), (5, 16), (100, 33), (7, 64), (3, 290)):
        part = (case[0][lo:lo + n], case[1][lo:lo + n]) + case[2:]
        assert torch.equal(_run(w4a8, part, "fp32"), whole[lo:lo + n])


def test_outputs_of_odd_address_and_pitch(w4a8, cuda):
    case = _case(21, 77, 224, 8)
    for dtype in DTYPES:
        Y = torch.zeros(21 * 81 + 1, device=cuda).to(DTYPES[dtype])[1:].view(21, 81)
        w4a8.launch_gemm_w8a8(*case[:4], Y, 81, 21, 77, 224, dtype, bias=case[4])
        assert torch.equal(Y[:, :77], _want(*case, dtype)) and (Y[:, 77:] == 0).all()


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("S,K", [(1, 32), (3, 5120), (200, 416), (2, 32768), (150, 8224), (17, 16384)])
def test_rows_are_quantized_by_the_definition(w4a8, cuda, S, K, dtype):
    g = torch.Generator(device="cuda").manual_seed(K)
    x = (torch.randn(S, K + 8, generator=g, device=cuda) * torch.exp(2 * torch.randn(S, 1, generator=g, device=cuda))).to(DTYPES[dtype])
    x[S // 2] = 0
    xq, xs = torch.full((S + 1, K), 9, dtype=torch.int8, device=cuda), torch.full((S + 1,), 9.0, device=cuda)
    w4a8.launch_quantize_rows_q8(x, K + 8, S, K, xq, xs, dtype)
    q, scale, _ = quantize(x[:, :K].float(), 0)
    assert torch.equal(xq[:S], q) and torch.equal(xs[:S], scale[:, 0]) and (xq[S] == 9).all() and xs[S] == 9


@pytest.mark.parametrize("M,N,K", [(1, 640, 512), (16, 3000, 2048), (70, 128, 1024), (300, 600, 512)])
def test_weights_quantized_just_before_their_product(w4a8, cuda, M, N, K):
    """Rows and weights quantized on the same stream directly in front of the product, in both orders, many times over: what is fetched early is not stale."""
    g = torch.Generator(device="cuda").manual_seed(1)
    xq, xs = torch.empty(M, K, dtype=torch.int8, device=cuda), torch.empty(M, device=cuda)
    wq, ws = torch.empty(N, K, dtype=torch.int8, device=cuda), torch.empty(N, device=cuda)
    xw = [(torch.randn(M, K, generator=g, device=cuda), torch.randn(N, K, generator=g, device=cuda)) for _ in range(6)]
    Y = [torch.empty(M, N, device=cuda) for _ in xw]
    for i, ((x, w), y) in enumerate(zip(xw, Y)):
        if i % 2:
            w4a8.launch_quantize_rows_q8(w, K, N, K, wq, ws)
            w4a8.linear_w8a8(x, K, xq, xs, wq, ws, y, N, M, N, K)
        else:
            w4a8.launch_quantize_rows_q8(x, K, M, K, xq, xs)
            w4a8.launch_quantize_rows_q8(w, K, N, K, wq, ws)
            w4a8.linear_w8a8(None, K, xq, xs, wq, ws, y, N, M, N, K, skip_quantize=1)
    for (x, w), y in zip(xw, Y):
        (q, s, _), (p, t, _) = quantize(x, 0), quantize(w, 0)
        assert torch.equal(y, _want(q, s[:, 0], p, t[:, 0], None, "fp32"))


def test_two_streams_and_a_graph(w4a8, cuda):
    cases = [_case(40, 1000, 2048, 1), _case(500, 1000, 512, 2)]
    Y = [torch.empty(c[0].shape[0], 1000, device=cuda) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        for c, y, st in zip(cases, Y, streams):
            w4a8.launch_gemm_w8a8(*c[:4], y, 1000, c[0].shape[0], 1000, c[0].shape[1], bias=c[4], stream=st)
    torch.cuda.synchronize()
    for c, y in zip(cases, Y):
        assert torch.equal(y, _want(*c, "fp32"))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for c, y in zip(cases, Y):
            w4a8.launch_gemm_w8a8(*c[:4], y, 1000, c[0].shape[0], 1000, c[0].shape[1], bias=c[4])
    for c in cases:
        c[0].neg_()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for c, y in zip(cases, Y):
        assert torch.equal(y, _want(*c, "fp32"))
    w4a8.device_status()


@pytest.mark.parametrize("x_dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("M,N,K", [(1, 640, 32), (1, 17408, 5120), (2, 300, 416), (2, 4096, 4096), (1, 1000, 15360), (1, 129, 32768), (2, 5000, 1312), (3, 512, 1024), (1, 60000, 256), (2, 1, 96), (1, 40000, 6144)])
def test_a_row_or_two_in_one_call(w4a8, cuda, M, N, K, x_dtype):
    """linear_w8a8 of few rows, which the product may quantize itself: codes, scales and outputs are those of the two calls, for the caller's pitch, with nothing behind them."""
    g = torch.Generator(device="cuda").manual_seed(N + K)
    x = (torch.randn(M, K + 8, generator=g, device=cuda) * 3).to(DTYPES[x_dtype])
    if M > 1:
        x[1] = 0                                                          # a row of zeros
    _, _, wq, ws, b = _case(1, N, K, N)
    xq, xs = torch.full((M + 1, K), 99, dtype=torch.int8, device=cuda), torch.full((M + 1,), 7.0, device=cuda)
    q, scale, _ = quantize(x[:, :K].float(), 0)
    for y_dtype in ("fp32", "bf16"):
        Y = torch.full((M + 1, N + 3), 3.0, device=cuda).to(DTYPES[y_dtype])
        w4a8.linear_w8a8(x, K + 8, xq, xs, wq, ws, Y, N + 3, M, N, K, x_dtype, y_dtype, bias=b)
        assert torch.equal(xq[:M], q) and torch.equal(xs[:M], scale[:, 0]) and (xq[M] == 99).all() and xs[M] == 7
        assert torch.equal(Y[:M, :N], _want(q, scale[:, 0], wq, ws, b, y_dtype)) and (Y[M] == 3).all() and (Y[:, N:] == 3).all()
    w4a8.device_status()


def test_single_rows_at_the_ends_of_fp32(w4a8, cuda):
    """A row quantized by its product, of subnormal, huge, infinite elements and NaN, and of zeros: the two calls' bits."""
    N, K = 200, 512
    g = torch.Generator(device="cuda").manual_seed(6)
    base = torch.randn(1, K, generator=g, device=cuda)
    _, _, wq, ws, b = _case(1, N, K, 7)
    rows = [base * 1e-42, base * 1e-37, base * 1e37, base * 0, base.clone(), base.clone()]
    rows[4][0, 100], rows[5][0, 511] = float("inf"), float("nan")
    xq, xs, Y = torch.empty(1, K, dtype=torch.int8, device=cuda), torch.empty(1, device=cuda), torch.empty(1, N, device=cuda)
    xq2, xs2, Y2 = torch.empty_like(xq), torch.empty_like(xs), torch.empty_like(Y)
    for x in rows:
        w4a8.linear_w8a8(x, K, xq, xs, wq, ws, Y, N, 1, N, K, bias=b)
        w4a8.launch_quantize_rows_q8(x, K, 1, K, xq2, xs2)
        w4a8.launch_gemm_w8a8(xq2, xs2, wq, ws, Y2, N, 1, N, K, bias=b)
        assert torch.equal(xq, xq2) and torch.equal(xs.view(torch.int32), xs2.view(torch.int32)) and torch.equal(Y.isnan(), Y2.isnan()) and torch.equal(Y.nan_to_num(), Y2.nan_to_num())


def test_an_output_in_the_place_of_its_row(w4a8, cuda):
    """Y may be x's own memory: the row has been read before the outputs are written."""
    K = N = 2048
    x = torch.randn(1, K, device=cuda)
    _, _, wq, ws, _ = _case(1, N, K, 4, bias=False)
    q, scale, _ = quantize(x, 0)
    want = _want(q, scale[:, 0], wq, ws, None, "fp32")
    w4a8.linear_w8a8(x, K, torch.empty_like(q), torch.empty(1, device=cuda), wq, ws, x, N, 1, N, K)
    assert torch.equal(x, want)


def test_single_rows_in_a_chain_and_a_graph(w4a8, cuda):
    """Row after row through two matrices, each the next one's input: what a launch leaves is what the next one reads, also in a graph."""
    K = 1024
    mats = [_case(1, K, K, 20 + i, bias=False)[2:4] for i in range(2)]
    x = torch.randn(1, K, device=cuda)
    xq, xs = torch.empty(1, K, dtype=torch.int8, device=cuda), torch.empty(1, device=cuda)
    a, b = torch.empty(1, K, device=cuda), torch.empty(1, K, device=cuda)

    def chain():
        w4a8.linear_w8a8(x, K, xq, xs, *mats[0], a, K, 1, K, K)
        for _ in range(4):
            w4a8.linear_w8a8(a, K, xq, xs, *mats[1], b, K, 1, K, K)
            w4a8.linear_w8a8(b, K, xq, xs, *mats[0], a, K, 1, K, K)

    def plain(v):
        for m in [mats[0]] + [mats[1], mats[0]] * 4:
            q, s, _ = quantize(v, 0)
            v = _want(q, s[:, 0], *m, None, "fp32")
        return v
    chain()
    assert torch.equal(a, plain(x))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        chain()
    for seed in range(3):
        x.copy_(torch.randn(1, K, device=cuda))
        graph.replay()
        assert torch.equal(a, plain(x))
    w4a8.device_status()
