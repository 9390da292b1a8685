"""Weights of chosen experts whose scores are far below the largest one, or below what fp32 holds: renormalised, they are what 64 bits make of them."""
import numpy as np
import pytest
import torch

from test_gpu_moe_route import check, plain

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lead", [0.0, 30.0, 60.0, 90.0, 95.0, 104.0, 120.0, 300.0, 690.0])
def test_an_expert_that_is_shut_out_leads_the_chosen_ones(w4a8, cuda, lead):
    S, E = 50, 24
    g = torch.Generator(device="cuda").manual_seed(int(lead))
    logits = torch.randn(S, E, generator=g, device=cuda)
    logits[:, 5] += lead
    shut = torch.zeros(E, device=cuda)
    shut[5] = -float("inf")
    liked = torch.zeros(E, device=cuda)
    liked[[3, 11, 12, 20]] = torch.tensor([2.0, 2.5, 3.0, 3.5], device=cuda)
    for bias in (shut, liked):
        check(w4a8, logits, 4, bias=bias)
        check(w4a8, logits, 4, bias=bias, groups=4, topk_groups=3, group_score="max")
        check(w4a8, logits, 4, bias=bias, renormalise=False)


@pytest.mark.parametrize("middle", [-40.0, -60.0, -64.0, -80.0, -87.0, -89.0, -95.0, -104.0, -150.0, -700.0])
def test_sigmoids_that_fp32_does_not_hold(w4a8, cuda, middle):
    S, E = 50, 24
    g = torch.Generator(device="cuda").manual_seed(int(-middle))
    logits = middle + 2.0 * torch.randn(S, E, generator=g, device=cuda)
    check(w4a8, logits, 4, scoring="sigmoid")
    check(w4a8, logits, 4, scoring="sigmoid", scale=2.5)
    logits[:, ::3] = -3.0                                     # some ordinary scores among them
    check(w4a8, logits, 12, scoring="sigmoid")


def test_bare_sigmoids_down_to_the_smallest_number(w4a8, cuda):
    """Not renormalised: the score itself, also where it is subnormal."""
    logits = torch.linspace(-102.0, -60.0, 64, device=cuda)[None].contiguous()
    idx, weight = torch.empty(1, 32, dtype=torch.int32, device=cuda), torch.empty(1, 32, device=cuda)
    for lowest in (False, True):
        bias = None if not lowest else -torch.arange(64, dtype=torch.float32, device=cuda)      # the small ones chosen
        w4a8.launch_moe_route(w4a8.Router.of(64, 32, "sigmoid", bias, renormalise=False), logits, 64, 1, idx, weight)
        want_idx, want = plain(logits, 32, "sigmoid", bias, renormalise=False)
        # the exponential 2 ulp, 1 + e^-v and a quotient one each where they are taken; subnormal results are multiples of 2^-149
        assert np.array_equal(idx.cpu().numpy(), want_idx) and np.allclose(weight.cpu().numpy(), want, rtol=8 * 2.0 ** -24, atol=2 * 2.0 ** -149)
