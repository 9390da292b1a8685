"""Sigmoids near and below the smallest normal fp32 number (logits below about -87): experts and groups are still chosen as fp64 says."""
import numpy as np
import pytest
import torch

from test_gpu_moe_route import plain

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("middle", [-86.0, -87.2, -88.0, -95.0, -103.5, -120.0, -600.0])
@pytest.mark.parametrize("groups,topk_groups,score", [(1, 1, "max"), (4, 1, "sum2"), (4, 2, "sum2"), (8, 3, "max"), (8, 5, "sum2")])
def test_experts_of_tiny_scores(w4a8, cuda, groups, topk_groups, score, middle):
    S, E, topk = 400, 32, 3
    g = torch.Generator(device="cuda").manual_seed(int(-10 * middle) + groups)
    for spread in (0.3, 1e-4):
        logits = middle + spread * torch.randn(S, E, generator=g, device=cuda)
        idx, weight = torch.empty(S, topk, dtype=torch.int32, device=cuda), torch.empty(S, topk, device=cuda)
        w4a8.launch_moe_route(w4a8.Router.of(E, topk, "sigmoid", None, groups, topk_groups, score), logits, E, S, idx, weight)
        want, _ = plain(logits, topk, "sigmoid", None, groups, topk_groups, score)
        assert np.array_equal(idx.cpu().numpy(), want)
