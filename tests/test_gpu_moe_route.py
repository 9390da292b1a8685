"""The choice of experts (w4a8_moe_route) against the definition in 64 bits on the host: indices equal, ties to the lowest."""
import numpy as np
import pytest
import torch

from layer_plain import DTYPES

pytestmark = pytest.mark.gpu
MAX = float(np.finfo(np.float32).max)


def plain(logits, topk, scoring="softmax", bias=None, groups=1, topk_groups=1, group_score="max", renormalise=True, scale=1.0):
    x = np.nan_to_num(logits.float().cpu().numpy().astype(np.float64), nan=-np.inf, posinf=MAX, neginf=-np.inf)
    idx, weight = np.zeros((x.shape[0], topk), np.int32), np.zeros((x.shape[0], topk))
    b = np.zeros(x.shape[1]) if bias is None else bias.cpu().numpy().astype(np.float64)
    for t, v in enumerate(x):
        with np.errstate(over="ignore"):
            if scoring == "sigmoid":
                s = 1.0 / (1.0 + np.exp(-v))
            else:
                e = np.exp(v - (v.max() if v.max() > -np.inf else 0.0))
                s = e / e.sum() if e.sum() > 0 else e
        c = v if scoring == "softmax" and bias is None and (group_score == "max" or topk_groups == groups) else s + b
        open_ = np.ones(len(v), bool)
        if topk_groups < groups:
            m = np.sort(c.reshape(groups, -1), 1)
            score = m[:, -1] if group_score == "max" else m[:, -1] + m[:, -2]
            best = np.lexsort((np.arange(groups), -score))[:topk_groups]
            open_ = np.isin(np.arange(len(v)) // (len(v) // groups), best)
        order = np.lexsort((np.arange(len(v)), -c, ~open_))[:topk]
        w = s[order]
        idx[t], weight[t] = order, (w / w.sum() if renormalise and w.sum() > 0 else w) * np.float64(np.float32(scale))
    return idx, weight


def check(w4a8, logits, topk, dtype="fp32", **how):
    S, E = logits.shape
    router = w4a8.Router.of(E, topk, **how)
    idx = torch.full((S + 1, topk), -7, dtype=torch.int32, device=logits.device)
    weight = torch.full((S + 1, topk), -7.0, device=logits.device)
    w4a8.launch_moe_route(router, logits, logits.stride(0), S, idx, weight, dtype)
    want_idx, want = plain(logits, topk, **how)
    assert np.array_equal(idx[:S].cpu().numpy(), want_idx)
    # fp32: the exponential 2 ulp and, of its argument's rounding, |v| e^v < 0.4 of the largest weight; the sum of 32 (1024) terms 6 (38) roundings, two quotients, the scale
    assert np.allclose(weight[:S].cpu().numpy(), want, rtol=(54 if how.get("renormalise", True) is False else 22) * 2.0 ** -24, atol=2.0 ** -24 * 2.5)
    assert (idx[S] == -7).all() and (weight[S] == -7).all()


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("S,E,topk,groups,topk_groups,group_score", [
    (1, 8, 2, 1, 1, "max"), (3, 1, 1, 1, 1, "max"), (5, 60, 4, 1, 1, "max"), (4, 60, 6, 4, 3, "sum2"), (9, 128, 8, 1, 1, "max"), (130, 256, 8, 8, 4, "sum2"), (33, 160, 6, 8, 3, "max"),
    (6, 512, 16, 1, 1, "max"), (7, 1024, 32, 1, 1, "max"), (5, 1024, 10, 32, 7, "sum2"), (3, 33, 32, 1, 1, "max"), (2, 96, 3, 3, 1, "sum2"), (8, 64, 8, 32, 4, "sum2"), (4, 999, 9, 27, 5, "max"), (3, 1020, 20, 17, 9, "sum2")])
def test_experts_and_weights(w4a8, cuda, S, E, topk, groups, topk_groups, group_score, scoring, dtype):
    g = torch.Generator(device="cuda").manual_seed(S * E)
    logits = (1.5 * torch.randn(S, E + 3, generator=g, device=cuda)).to(DTYPES[dtype])[:, :E]         # rows of odd pitch; 16-bit logits have ties
    bias = 0.1 * torch.randn(E, generator=g, device=cuda)
    for b in (None, bias):
        for renormalise in (True, False):
            check(w4a8, logits, topk, dtype, scoring=scoring, bias=b, groups=groups, topk_groups=topk_groups, group_score=group_score, renormalise=renormalise, scale=2.5)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_ties_masks_and_numbers_that_are_none(w4a8, cuda, scoring):
    E, inf, nan = 64, float("inf"), float("nan")
    rows = torch.zeros(9, E, device=cuda)                              # row 0: all equal
    rows[1] = -inf                                                     # nothing is left
    rows[2] = torch.finfo(torch.float32).min
    rows[3, ::2] = -inf
    rows[4] = -inf
    rows[4, 40] = 3.0                                                  # one expert, the others chosen behind it by index
    rows[5, 7], rows[5, 9] = nan, 1.0
    rows[6, 5], rows[6, 50] = inf, inf
    rows[7] = nan
    rows[8, 1::2] = -0.0                                               # equal to 0
    for how in (dict(), dict(groups=8, topk_groups=3, group_score="sum2"), dict(bias=torch.linspace(-1, 1, E, device=cuda))):
        check(w4a8, rows, 6, scoring=scoring, **how)
        check(w4a8, rows, 6, scoring=scoring, renormalise=False, **how)
    check(w4a8, rows.half(), 6, "fp16", scoring=scoring)


def test_indices_are_experts_whatever_the_bias(w4a8, cuda):
    E, bias = 40, torch.randn(40, device=cuda)
    bias[3], bias[5], bias[8] = float("nan"), float("inf"), -float("inf")
    logits = torch.randn(50, E, device=cuda)
    idx, weight = torch.empty(50, 8, dtype=torch.int32, device=cuda), torch.empty(50, 8, device=cuda)
    w4a8.launch_moe_route(w4a8.Router.of(E, 8, "sigmoid", bias, 4, 3, "sum2"), logits, E, 50, idx, weight)
    got = idx.cpu().numpy()
    assert got.min() >= 0 and got.max() < E and all(len(set(r)) == 8 for r in got)


def test_many_tokens_two_streams_and_a_graph(w4a8, cuda):
    S, E = 3001, 128
    logits = [torch.randn(S, E, device=cuda) for _ in range(2)]
    router = w4a8.Router.of(E, 8)
    out = [(torch.empty(S, 8, dtype=torch.int32, device=cuda), torch.empty(S, 8, device=cuda)) for _ in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for st, l, o in zip(streams, logits, out):
            w4a8.launch_moe_route(router, l, E, S, *o, stream=st)
    torch.cuda.synchronize()
    for l, o in zip(logits, out):
        want_idx, want = plain(l, 8)
        assert np.array_equal(o[0].cpu().numpy(), want_idx) and np.allclose(o[1].cpu().numpy(), want, rtol=22 * 2.0 ** -24, atol=2.0 ** -24)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w4a8.launch_moe_route(router, logits[0], E, S, *out[0])
    logits[0].copy_(logits[1])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])
