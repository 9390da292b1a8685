"""The border between the last expert that is taken and the first that is not (w4a8_moe_route), with no room for candidates to spare: fp32 cannot tell
the experts on its two sides apart, the definition's fp64 can."""
import numpy as np
import pytest
import torch

from test_gpu_moe_route import check

pytestmark = pytest.mark.gpu


def rows_of(E, topk, at, ulps, seed, dev):
    """topk - 1 experts far ahead by their bias, the others within `ulps` steps of fp32 of `at`, in another order in each row."""
    rng = np.random.default_rng(seed)
    order = rng.permutation(E)
    ahead, near = order[:topk - 1], np.sort(order[topk - 1:])
    bias = np.zeros(E, np.float32)
    bias[ahead] = 1.0 + 0.01 * np.arange(1, topk)
    logits = np.zeros((64, E), np.float32)
    for row in logits:
        row[near] = np.float32(at) + rng.permutation(len(near)).astype(np.float32) * np.float32(ulps) * np.spacing(np.float32(at))
    return torch.from_numpy(logits).to(dev), torch.from_numpy(bias).to(dev)


def test_two_scores_that_are_one_fp32_number(w4a8, cuda):
    """33 experts: 31 far ahead, and of the two that are left the second one's logit is the next fp32 number."""
    bias = torch.zeros(33, device=cuda)
    bias[2:] = 1.0 + 0.01 * torch.arange(1, 32, device=cuda)
    logits = torch.zeros(1, 33, device=cuda)
    logits[0, 0] = 8.0
    logits[0, 1] = float(np.nextafter(np.float32(8.0), np.float32(9.0)))
    check(w4a8, logits, 32, scoring="sigmoid", bias=bias)


@pytest.mark.parametrize("scoring,at", [("sigmoid", 8.0), ("sigmoid", 0.5), ("softmax", 1.0)])
@pytest.mark.parametrize("topk", [16, 28, 29, 31, 32])
@pytest.mark.parametrize("E", [33, 36, 64, 250, 1024])
def test_the_last_expert_taken(w4a8, cuda, E, topk, scoring, at):
    for ulps in (1, 3):
        logits, bias = rows_of(E, topk, at, ulps, E + topk, cuda)
        check(w4a8, logits, topk, scoring=scoring, bias=bias)


@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_the_last_expert_of_open_groups(w4a8, cuda, scoring):
    for seed in range(4):
        logits, bias = rows_of(96, 32, 2.0, 1, seed, cuda)
        for score in ("max", "sum2"):
            check(w4a8, logits, 32, scoring=scoring, bias=bias, groups=8, topk_groups=5, group_score=score)


@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_equal_choices_and_nothing_left(w4a8, cuda, scoring):
    """Choices that are equal in fp64 too go to the lowest index; 32 of 32 experts leave no border."""
    logits, bias = rows_of(40, 32, 3.0, 0, 1, cuda)
    check(w4a8, logits, 32, scoring=scoring, bias=bias)
    logits, bias = rows_of(32, 32, 3.0, 1, 2, cuda)
    check(w4a8, logits, 32, scoring=scoring, bias=bias)
    check(w4a8, logits, 32, scoring=scoring, bias=torch.zeros_like(bias))
