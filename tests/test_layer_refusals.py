"""What the layer operators refuse, before any device work: runs without a GPU."""
import ctypes

import pytest
import torch

GPU = torch.cuda.is_available()      # the pointers are made up: calls that are allowed get as far as the device check, without a device
P = lambda n: ctypes.c_void_p(n)
BASE = 1 << 20


def code(w4a8, rc, text):
    assert text in w4a8.lib().w4a8_last_error(), w4a8.lib().w4a8_last_error()
    return rc


def norm_of(w4a8, **more):
    n = w4a8.Norm(BASE, BASE + 4096, None, 0, 1e-6, 1.0, 64, 0, -1, 0, 0)
    for k, v in more.items():
        setattr(n, k, v)
    return n


def add_norm(w4a8, n, h=BASE << 1, ldh=64, y=BASE << 2, ldy=64, ho=None, ldo=64, no=BASE << 3, ldn=64, xq=None, xs=None, xsum=None, group=32, S=4):
    return w4a8.lib().w4a8_add_norm(n, P(h), ldh, P(y), ldy, P(ho), ldo, P(no), ldn, P(xq), P(xs), P(xsum), group, S, None)


def test_add_norm(w4a8):
    A, L, U = w4a8.ERR_ARG, w4a8.ERR_ALIGN, w4a8.ERR_UNSUPPORTED
    N = lambda **k: norm_of(w4a8, **k)
    bad = [(N(K=48), {}, A, b"multiple of 32"), (N(K=-32), {}, A, b"multiple"), (N(K=32800), dict(ldh=32800, ldy=32800, ldn=32800), U, b"at most"), (N(dtype=3), {}, A, b"dtype"),
           (N(dtype=0, y_dtype=1), {}, A, b"y_dtype"), (N(dtype=1, y_dtype=2), {}, A, b"y_dtype"), (N(variant=3), {}, A, b"variant"), (N(variant=-2), {}, A, b"variant"),
           (N(post_variant=4), {}, A, b"variant"), (N(eps=-1.0), {}, A, b"eps"), (N(eps=float("nan")), {}, A, b"eps"), (N(), dict(group=16), A, b"group"), (N(), dict(S=-1), A, b"S=-1"),
           (N(), dict(h=None), A, b"null"), (N(weight=None), {}, A, b"null"), (N(post_variant=1, post_weight=None), {}, A, b"null"), (N(), dict(no=None), A, b"no output"),
           (N(), dict(xq=BASE << 4), A, b"null"), (N(), dict(xs=BASE << 4), A, b"without xq"), (N(), dict(xq=BASE << 4, xs=BASE << 5, xsum=BASE << 6, group=0), A, b"no xsum"),
           (N(), dict(ldh=60), A, b"pitch"), (N(), dict(ldy=32), A, b"pitch"), (N(), dict(ldn=0), A, b"pitch"), (N(), dict(ldh=66), L, b"16-byte"), (N(), dict(h=BASE + 4), L, b"16-byte"),
           (N(), dict(y=(BASE << 2) + 8), L, b"16-byte"), (N(), dict(no=(BASE << 3) + 2), L, b"16-byte"), (N(weight=BASE + 4), {}, L, b"weights"), (N(gate=BASE + 8), {}, L, b"gate"),
           (N(gate=BASE, gate_ld=32), {}, A, b"gate"), (N(), dict(xq=(BASE << 4) + 4, xs=BASE << 5), L, b"xq"),
           # overlaps: an output over an input it may not replace, shifted rows, other pitch, two outputs, weights
           (N(), dict(no=(BASE << 1) + 64), A, b"overlaps"), (N(), dict(ho=BASE << 2), A, b"h_out overlaps y"), (N(), dict(no=BASE << 1, ldn=128), A, b"overlaps"),
           (N(), dict(ho=BASE << 3), A, b"n_out overlaps h_out"), (N(), dict(no=BASE), A, b"weight"), (N(dtype=1, y_dtype=0), dict(no=BASE << 2), A, b"overlaps"),
           (N(), dict(xq=BASE << 1, xs=BASE << 5), A, b"xq overlaps h"), (N(), dict(xq=BASE << 4, xs=(BASE << 4) + 16), A, b"xs overlaps xq")]
    for n, args, want, text in bad:
        assert code(w4a8, add_norm(w4a8, n, **args), text) == want, (args, text)
    assert add_norm(w4a8, N(), S=0, h=None) == w4a8.OK
    assert add_norm(w4a8, None) == A
    for args in () if GPU else (dict(no=BASE << 1), dict(no=BASE << 2), dict(ho=BASE << 1), dict(ldh=128, no=(BASE << 1) + 256, ldn=128), dict(xq=BASE << 4, xs=BASE << 5, group=0)):
        assert add_norm(w4a8, N(), **args) not in (A, L), args


def test_quantize_rows(w4a8):
    f = w4a8.lib().w4a8_quantize_rows_q8
    assert f(None, 64, 4, 64, 0, P(BASE), P(BASE), None) == w4a8.ERR_ARG
    assert f(P(BASE << 1), 64, 4, 64, 5, P(BASE), P(BASE << 2), None) == w4a8.ERR_ARG
    assert f(P(BASE << 1), 64, 4, 40, 0, P(BASE), P(BASE << 2), None) == w4a8.ERR_ARG
    assert f(P(BASE << 1), 64, 4, 64, 0, P(BASE << 1), P(BASE << 2), None) == w4a8.ERR_ARG
    assert f(P(BASE << 1), 65536, 4, 65536, 0, P(BASE), P(BASE << 2), None) == w4a8.ERR_UNSUPPORTED
    assert f(None, 64, 0, 64, 0, None, None, None) == w4a8.OK


def rope_qk(w4a8, r, q=BASE, ldq=512, hq=4, k=BASE + 1024, ldk=512, hk=2, position=BASE << 1, T=3, qo=BASE << 2, ldqo=256, ko=BASE << 3, ldko=128, dtype=0):
    return w4a8.lib().w4a8_rope_qk(r, P(q), ldq, hq, P(k), ldk, hk, P(position), T, P(qo), ldqo, P(ko), ldko, dtype, None)


def test_rope(w4a8):
    A, L = w4a8.ERR_ARG, w4a8.ERR_ALIGN

    def R(**more):
        r = w4a8.Rope(BASE << 4, BASE << 5, BASE << 6, 1e-6, 1.0, 64, 64, 0, 0)
        for k, v in more.items():
            setattr(r, k, v)
        return r
    bad = [(R(dim=60), {}, A, b"dim"), (R(dim=0), {}, A, b"dim"), (R(dim=264), {}, A, b"dim"), (R(rotary=12), {}, A, b"rotary"), (R(rotary=72), {}, A, b"rotary"), (R(rotary=-8), {}, A, b"rotary"),
           (R(variant=3), {}, A, b"variant"), (R(eps=-1.0), {}, A, b"eps"), (R(), dict(dtype=3), A, b"dtype"), (R(), dict(T=-1), A, b"T=-1"), (R(), dict(hq=-1), A, b"heads_q"),
           (R(), dict(hk=70000), A, b"heads_k"), (R(turns=None), {}, A, b"null"), (R(q_weight=None), {}, A, b"null"), (R(k_weight=None), {}, A, b"null"), (R(), dict(position=None), A, b"null"),
           (R(), dict(q=None), A, b"null"), (R(), dict(ko=None), A, b"null"), (R(), dict(ldq=128), A, b"pitch"), (R(), dict(ldko=64), A, b"pitch"), (R(), dict(q=BASE + 4), L, b"16-byte"),
           (R(), dict(ldqo=258), L, b"16-byte"), (R(k_weight=BASE + 4), {}, L, b"weights"), (R(turns=BASE + 4), {}, L, b"turns"), (R(), dict(qo=BASE + 256), A, b"overlaps"),
           (R(), dict(qo=BASE, ldqo=1024), A, b"overlaps"), (R(), dict(qo=BASE << 3), A, b"k_out overlaps q_out"), (R(), dict(ko=BASE << 1), A, b"position")]
    for r, args, want, text in bad:
        assert code(w4a8, rope_qk(w4a8, r, **args), text) == want, (args, text)
    assert rope_qk(w4a8, None) == A
    assert rope_qk(w4a8, R(), T=0, q=None) == w4a8.OK
    for args in () if GPU else (dict(qo=BASE, ldqo=512, ko=BASE + 1024, ldko=512), dict(hk=0, k=None, ko=None, ldk=0, ldko=0), {}):
        assert rope_qk(w4a8, R(), **args) not in (A, L), args


def test_moe_route(w4a8):
    A = w4a8.ERR_ARG

    def call(bias=None, experts=64, topk=4, scoring=0, groups=1, topk_groups=1, group_score=0, logits=BASE, ld=64, S=3, dtype=0, idx=BASE << 1, weight=BASE << 2):
        r = w4a8.Router(bias, experts, topk, scoring, groups, topk_groups, group_score, 1, 1.0)
        return w4a8.lib().w4a8_moe_route(r, P(logits), ld, S, dtype, P(idx), P(weight), None)
    for args in (dict(experts=0), dict(experts=1025, ld=1025), dict(topk=0), dict(topk=33), dict(groups=0), dict(groups=33, experts=66, ld=66), dict(groups=5), dict(groups=4, topk_groups=5),
                 dict(groups=4, topk_groups=0), dict(groups=32, topk_groups=1, topk=4), dict(scoring=2), dict(group_score=2), dict(ld=63), dict(S=-1), dict(dtype=4), dict(logits=None),
                 dict(idx=None), dict(weight=None), dict(idx=BASE), dict(weight=BASE << 1), dict(bias=BASE << 2), dict(experts=8, ld=8, topk=2, groups=8, topk_groups=4, group_score=1)):
        assert call(**args) == A, args
    assert call(logits=BASE + 2) == w4a8.ERR_ALIGN
    assert call(S=0, logits=None) == w4a8.OK
    assert w4a8.lib().w4a8_moe_route(None, P(BASE), 64, 1, 0, P(BASE), P(BASE), None) == A


def test_gemm_w8a8(w4a8):
    A = w4a8.ERR_ARG

    def call(xq=BASE, xs=BASE << 1, wq=BASE << 2, ws=BASE << 3, bias=None, Y=BASE << 4, ldy=40, M=8, N=40, K=64, dtype=0):
        return w4a8.lib().w4a8_gemm_w8a8(P(xq), P(xs), P(wq), P(ws), P(bias), P(Y), ldy, M, N, K, dtype, None)
    for args in (dict(M=-1), dict(N=-1), dict(K=48), dict(K=0), dict(K=-32), dict(dtype=3), dict(xq=None), dict(xs=None), dict(wq=None), dict(ws=None), dict(Y=None), dict(ldy=39), dict(Y=BASE + 256),
                 dict(Y=BASE << 1), dict(bias=(BASE << 4) + 4)):
        assert call(**args) == A, args
    assert call(K=131072) == w4a8.ERR_UNSUPPORTED
    assert call(M=2 ** 31 - 1023) == w4a8.ERR_UNSUPPORTED and call(N=2 ** 31 - 1, ldy=2 ** 31) == w4a8.ERR_UNSUPPORTED
    for args in (dict(xq=BASE + 8), dict(wq=(BASE << 2) + 4), dict(Y=(BASE << 4) + 2)):
        assert call(**args) == w4a8.ERR_ALIGN, args
    assert call(M=0, xq=None) == w4a8.OK and call(N=0, ldy=0, Y=None) == w4a8.OK
    assert w4a8.lib().w4a8_linear_w8a8(None, 64, P(BASE), P(BASE << 1), P(BASE << 2), P(BASE << 3), None, P(BASE << 4), 40, 8, 40, 64, 0, 0, 0, None) == A
    assert w4a8.lib().w4a8_linear_w8a8(P(BASE << 5), 64, P(BASE), P(BASE << 1), P(BASE << 2), P(BASE << 3), None, P(BASE << 4), 40, -1, 40, 64, 0, 0, 0, None) == A


def test_structs_of_tensors(w4a8):
    with pytest.raises(ValueError):
        w4a8.Norm.of(64, torch.zeros(64))                    # not on a GPU
    with pytest.raises(ValueError):
        w4a8.Rope.of(64, 64, q_weight=torch.zeros(64), k_weight=torch.zeros(64), device="cpu")
    with pytest.raises(ValueError):
        w4a8.Router.of(64, 8, bias=torch.zeros(63))
    with pytest.raises(KeyError):
        w4a8.Router.of(64, 8, scoring="sparse")


def test_the_binding_without_ctypes(w4a8):
    """The launchers' own way into the library: what it cannot convert is an exception, what the library refuses is its error."""
    t = torch.zeros(4, 64, device="cuda" if GPU else "cpu")
    n = norm_of(w4a8, K=48)
    with pytest.raises(w4a8.W4A8Error, match="multiple of 32") as e:
        w4a8.launch_add_norm(n, t, t, 4, N=t, stream=0)
    assert e.value.code == w4a8.ERR_ARG
    with pytest.raises(w4a8.W4A8Error, match="no output"):
        w4a8.launch_add_norm(norm_of(w4a8), t, None, 4, stream=0)
    with pytest.raises(w4a8.W4A8Error, match="pitch"):
        w4a8.launch_gemm_w8a8(t, t, t, t, t, 39, 8, 40, 64, stream=0)
    with pytest.raises(w4a8.W4A8Error, match="null"):
        w4a8.linear_w8a8(None, 64, t, t, t, t, t, 40, 8, 40, 64, stream=0)
    with pytest.raises(w4a8.W4A8Error, match="null"):
        w4a8.launch_quantize_rows_q8(t, 64, 4, 64, t, None, stream=0)
    with pytest.raises(w4a8.W4A8Error, match="experts"):
        w4a8.launch_moe_route(w4a8.Router.of(64, 40), t, 64, 4, t, t, stream=0)
    with pytest.raises(w4a8.W4A8Error, match="dtype"):
        w4a8.launch_rope_qk(w4a8.Rope(), t, 64, 1, t, 64, 1, t, 4, dtype=7, stream=0)
    w4a8.launch_add_norm(norm_of(w4a8), None, None, 0, stream=0)                     # nothing to do
    with pytest.raises(OverflowError):
        w4a8.launch_add_norm(norm_of(w4a8), t, t, 1 << 40, N=t, stream=0)
    with pytest.raises(TypeError):
        w4a8.launch_add_norm(norm_of(w4a8), t, t, 4.0, N=t, stream=0)
    with pytest.raises(AttributeError):
        w4a8.launch_add_norm(norm_of(w4a8), "h", t, 4, N=t, stream=0)
    with pytest.raises(TypeError, match="a struct of"):
        w4a8._binding().add_norm(w4a8.Rope(), t, 64, t, 64, None, 64, t, 64, None, None, None, 32, 4, 0)
    n = norm_of(w4a8)
    n._gate_rows = 3                                         # what Norm.of notes of a gate with a row for each token
    with pytest.raises(ValueError, match="4 rows, a gate of 3"):
        w4a8.launch_add_norm(n, t, t, 4, N=t, stream=0)
    with pytest.raises(TypeError, match="15 expected"):
        w4a8._binding().add_norm(norm_of(w4a8), t)


class Elsewhere:
    """What the binding looks at of a tensor on another GPU than the current one, which is 0 here."""
    is_cuda = True

    def __init__(self, gpu):
        self.gpu = gpu

    def get_device(self):
        return self.gpu

    def data_ptr(self):
        return BASE


def test_tensors_that_are_not_on_the_current_gpu(w4a8):
    """A kernel would follow their pointers; where there is no GPU at all, nothing is launched.  The calls here have no rows."""
    b, t = w4a8._binding(), torch.zeros(4, 64)
    n = norm_of(w4a8)
    try:
        for gpus, kind in ((1, torch.Tensor), (2, torch.Tensor), (1, Elsewhere), (2, None)):          # the tensors' type as torch's and as anybody's
            b.streams(lambda: 0, lambda device: 0, gpus, kind)
            with pytest.raises(ValueError, match="not on a GPU"):
                w4a8.launch_add_norm(n, t, None, 0, N=None, stream=0)
            with pytest.raises(ValueError, match="not on a GPU"):
                w4a8.launch_gemm_w8a8(None, None, t, None, None, 64, 0, 64, 64, stream=0)
            w4a8.launch_add_norm(n, Elsewhere(0), None, 0, stream=0)
            w4a8.launch_add_norm(n, BASE, None, 0, stream=0)                          # a number is the caller's word
        with pytest.raises(ValueError, match="on GPU 1, the current one is 0"):
            w4a8.launch_add_norm(n, Elsewhere(1), None, 0, stream=0)
        with pytest.raises(AttributeError):
            w4a8.launch_add_norm(n, "h", None, 0, stream=0)
    finally:
        w4a8._native = None                                  # bound anew with torch's own functions
    with pytest.raises(ValueError, match="table is not on a GPU"):
        w4a8.launch_rope_qk(w4a8.Rope.of(64, 64, device="cpu"), BASE, 64, 1, BASE << 1, 64, 1, BASE << 2, 0, stream=0)
