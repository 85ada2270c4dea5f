"""Masked experts of a router with a bias: what the documentation says of them, case by case."""
import math

import pytest
import torch

from kaillm_b200 import linear
from tests.gpu_util import dev

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("mask", [-math.inf, math.nan])
def test_a_masked_expert_counts_with_its_bias(scoring, dtype, mask):
    x = torch.tensor([[0.0, mask, 1.0, mask]], dtype=dtype, device=dev())
    b = torch.tensor([0.0, 1.5, 0.0, -0.5], device=dev())
    w, ids = linear.route_experts(x, 3, scoring=scoring, bias=b)
    assert ids.tolist() == [[1, 2, 0]] and w[0, 0] == 0 and abs(float(w.sum()) - 1) < 1e-6 and bool((w[0, 1:] > 0).all())
    w, ids = linear.route_experts(x, 1, scoring=scoring, bias=b)
    assert ids.tolist() == [[1]] and w.tolist() == [[0.0]]
    assert linear.route_experts(x, 4, scoring=scoring)[1].tolist() == [[2, 0, 1, 3]]              # without a bias: last, in their order


@pytest.mark.parametrize("experts,groups,top_groups", [(64, 1, 1), (256, 1, 1), (60, 1, 1), (1024, 1, 1), (256, 8, 4), (96, 3, 2), (32, 4, 2)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("mask", [-math.inf, math.nan])
def test_a_bias_of_minus_infinity_places_an_expert_last(scoring, experts, groups, top_groups, mask):
    """Half of every group out by logit and bias, half of those by the bias alone: none of them is chosen while others are left."""
    g = torch.Generator().manual_seed(experts)
    x = torch.randn((33, experts), generator=g)
    b = torch.randn(experts, generator=g) * 0.3
    out = torch.arange(experts) % 2 == 1
    b[out] = mask
    x[:, torch.arange(experts) % 4 == 1] = mask
    w, ids = linear.route_experts(x.to(dev()), 5, scoring=scoring, bias=b.to(dev()), groups=groups, top_groups=top_groups)
    assert not bool(out[ids.cpu().long()].any()) and bool((w > 0).all()) and all(len(set(r)) == 5 for r in ids.tolist())
