"""Scores that fp32 cannot tell apart, where its errors are largest: sums of large biases that cancel, and a thousand experts."""
import pytest
import torch

from kaillm_b200 import linear
from tests.attention_util import route
from tests.gpu_util import dev

pytestmark = pytest.mark.gpu


def same_ids(x, k, scoring, bias, groups, top_groups):
    got = linear.route_experts(x.to(dev()), k, scoring=scoring, bias=bias.to(dev()), groups=groups, top_groups=top_groups)[1].cpu()
    assert torch.equal(got, route(x, k, scoring, bias, groups, top_groups, True, 1.0)[1])


@pytest.mark.parametrize("experts,groups,top_groups", [(32, 4, 2), (64, 4, 2), (128, 8, 3), (96, 3, 1), (60, 5, 2), (256, 8, 4)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("large", [1000.0, 30.0])
def test_large_biases_that_cancel_in_a_group(experts, groups, top_groups, scoring, large):
    """A group's best two stand at p + large and p - large, rounded to steps of `large`; their sum is near zero and the groups' sums are
    apart by less than that."""
    size, g = experts // groups, torch.Generator().manual_seed(experts)
    x = torch.randn((200, experts), generator=g) * 0.01
    bias = torch.full((experts,), -10 * large)
    first = torch.arange(groups) * size
    bias[first], bias[first + size - 1] = large, -large
    x[:, first] = torch.randn((200, groups), generator=g) * large * 2.0 ** -22
    same_ids(x, 2, scoring, bias, groups, top_groups)


@pytest.mark.parametrize("experts", [1024, 1000, 700])
@pytest.mark.parametrize("top", [0.0, 5.0])
@pytest.mark.parametrize("k", [4, 15, 32])
def test_a_thousand_close_scores(experts, top, k):
    """Softmax with a bias, no groups: one expert ahead of the others (whose sum is then as large as its own term) or none; biases that
    bring many scores together to a few steps of fp32."""
    g = torch.Generator().manual_seed(experts + k)
    x = torch.randn((40, experts), generator=g) * 0.3
    x[:, 17] += top
    p = torch.softmax(x[0].double(), -1)
    bias = (p.max() - p).float()                      # for the first token all scores are the same but for the rounding of the bias
    x[1:] = x[0] + torch.randn((39, experts), generator=g) * 2.0 ** -22
    same_ids(x, k, "softmax", bias, 1, 1)
