"""Routing of tokens to experts against 64 bits with Python's sorting, and in front of the experts' products."""
import math

import pytest
import torch

from kaillm_b200 import linear
from tests.attention_util import DT, route
from tests.gpu_util import act, dev
from tests.test_moe_gpu import experts_wire

pytestmark = pytest.mark.gpu


def check(logits, top_k, scoring="softmax", bias=None, groups=1, top_groups=1, renormalize=True, scale=1.0):
    w, ids = linear.route_experts(logits, top_k, scoring=scoring, bias=bias, groups=groups, top_groups=top_groups, renormalize=renormalize, scale=scale)
    want_w, want_ids = route(logits, top_k, scoring, bias, groups, top_groups, renormalize, scale)
    assert w.dtype == torch.float32 and ids.dtype == torch.int32 and torch.equal(ids.cpu(), want_ids)
    # a probability: the difference to the maximum rounded once (half a step of up to 2^7 for the logits used here: 2^-17), the
    # exponential 2 ulp, the sum of E terms; the renormalised weight: twice that and a sum of 32
    tol = 2 * (2.0 ** -17 + 2.0 ** -22 + logits.shape[1] * 2.0 ** -24) + 40 * 2.0 ** -24
    assert bool(((w.cpu().double() - want_w).abs() <= tol * want_w + 1e-37).all())
    return w, ids


def logits(t, e, dtype, seed=0, spread=2.0):
    return (torch.randn((t, e), generator=torch.Generator().manual_seed(seed)) * spread).to(DT[dtype]).to(dev())


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("t,e,k", [(1, 1, 1), (5, 8, 2), (7, 60, 4), (64, 64, 6), (33, 128, 8), (9, 160, 6), (100, 256, 8), (3, 384, 10), (17, 512, 32), (4, 1024, 32),
                                   (1, 33, 32)])
def test_sizes(dtype, scoring, t, e, k):
    check(logits(t, e, dtype, seed=e), k, scoring)
    check(logits(t, e, dtype, seed=e), k, scoring, bias=torch.randn(e, device=dev()) * 0.2, renormalize=False, scale=2.5)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("e,groups,top_groups,k", [(256, 8, 4, 8), (64, 4, 1, 6), (160, 8, 3, 6), (32, 32, 8, 8), (96, 3, 2, 5), (1024, 32, 32, 4), (12, 2, 2, 12)])
def test_groups(scoring, bias, e, groups, top_groups, k):
    b = torch.randn(e, device=dev()) * 0.1 if bias else None
    check(logits(50, e, "f32", seed=e), k, scoring, b, groups, top_groups)


@pytest.mark.parametrize("groups", [1, 4])
def test_ties_go_to_the_lowest_index(groups):
    x = torch.randint(0, 3, (40, 64), generator=torch.Generator().manual_seed(0)).float().to(dev())
    check(x, 8, groups=groups, top_groups=max(1, groups // 2))
    check(x, 8, "sigmoid", torch.zeros(64, device=dev()), groups=groups, top_groups=max(1, groups // 2))
    check(torch.zeros((2, 64), device=dev()), 8, groups=groups, top_groups=max(1, groups // 2))
    zero = torch.zeros((1, 64), device=dev())
    zero[0, ::2] = -0.0
    check(zero, 8, groups=groups, top_groups=max(1, groups // 2))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
def test_masked_and_strange_logits(dtype, scoring, bias):
    x = logits(8, 64, dtype)
    x[0, :60] = -math.inf                    # fewer experts than top_k are left
    x[1] = -math.inf
    x[2, 5] = math.nan
    x[3, 7] = math.inf
    x[4, 1::2] = torch.finfo(DT[dtype]).min
    x[5] = math.nan
    b = torch.randn(64, device=dev()) * 0.1 if bias else None
    w, ids = check(x, 8, scoring, b)
    assert bool(torch.isfinite(w).all()) and all(len(set(r)) == 8 for r in ids.tolist())
    check(x, 6, scoring, b, groups=4, top_groups=2)


def test_scores_closer_than_fp32_tells_apart():
    """Sums of a sigmoid and a bias that agree in fp32: the choice is that of 64 bits, in every order of the experts."""
    x = torch.full((6, 40), -3.0, device=dev())
    bias = torch.zeros(40, device=dev())
    for r in range(6):
        x[r, 3 + r], x[r, 20 + r], x[r, 30 + r] = 2.0, 2.0 + 2.0 ** -22, 2.0 - 2.0 ** -22
    check(x, 2, "sigmoid", bias)
    check(x, 2, "softmax", bias)
    y = torch.full((4, 64), 17.0, device=dev())
    y[:, 5::8] += torch.arange(8, device=dev()) * 2.0 ** -18        # sigmoid(17 + d): 1 in fp32
    check(y, 5, "sigmoid", torch.zeros(64, device=dev()))
    check(y, 4, "sigmoid", torch.zeros(64, device=dev()), groups=8, top_groups=3)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("e,groups", [(256, 8), (128, 4), (512, 32), (96, 3), (64, 8), (1024, 16)])
def test_groups_closer_than_fp32_tells_apart(scoring, e, groups):
    """The best two of all groups the same but for single bits of one logit, in every order; then the same among the experts of one group."""
    size, g = e // groups, torch.Generator().manual_seed(e)
    x = torch.randn((64, e), generator=g) - 4
    for r in range(64):
        best = (torch.arange(groups) * size)[:, None] + torch.randint(0, size - 1, (groups, 1), generator=g) + torch.tensor([0, 1])
        x[r, best] = torch.tensor([1.0, 0.5])
        x[r, best[:, 0]] += torch.randint(-2, 3, (groups,), generator=g) * 2.0 ** -23
        x[r, :size] = 0.25 + torch.randint(-2, 3, (size,), generator=g) * 2.0 ** -24
    bias = torch.full((e,), 0.125, device=dev())
    check(x.to(dev()), 5, scoring, bias, groups, (groups + 1) // 2)
    check(x.to(dev()), 5, scoring, bias)
    check(x[:, :size].contiguous().to(dev()), 3, scoring, bias[:size])


def test_many_tokens_strides_and_capture():
    x = logits(3001, 256, "f32", seed=9)
    bias = torch.randn(256, device=dev()) * 0.05
    w, ids = check(x, 8, "sigmoid", bias, 8, 4, scale=2.5)
    wide = torch.zeros((3001, 300), device=dev())
    wide[:, 3:259] = x
    # rows that no vector load may touch take another kernel, whose sums have another order: compared with 64 bits as well
    assert torch.equal(check(wide[:, 3:259], 8, "sigmoid", bias, 8, 4, scale=2.5)[1], ids)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = linear.route_experts(x, 8, scoring="sigmoid", bias=bias, groups=8, top_groups=4, scale=2.5)
    x.copy_(x.flip(0).clone())
    graph.replay()
    assert torch.equal(got[0], w.flip(0)) and torch.equal(got[1], ids.flip(0))
    empty = linear.route_experts(x[:0], 8)
    assert empty[0].shape == (0, 8) and empty[1].shape == (0, 8)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("e,k,groups,top_groups", [(8, 2, 1, 1), (24, 4, 1, 1), (32, 4, 8, 3), (60, 6, 1, 1), (64, 8, 4, 2), (96, 5, 3, 1), (128, 15, 1, 1), (160, 6, 1, 1),
                                                   (256, 8, 1, 1), (256, 1, 8, 1), (256, 8, 2, 1)])
def test_many_tokens(dtype, scoring, e, k, groups, top_groups):
    """More tokens than a warp takes one by one, with an odd one at the end."""
    x = logits(1501, e, dtype, seed=e + k)
    check(x, k, scoring, None, groups, top_groups)
    check(x, k, scoring, torch.randn(e, device=dev()) * 0.1, groups, top_groups, renormalize=False, scale=0.5)


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("groups", [1, 4])
def test_many_tokens_with_ties_and_masks(bias, groups):
    x = torch.randint(0, 4, (1300, 64), generator=torch.Generator().manual_seed(1)).float().to(dev())
    x[100:200] = 0.0                         # more candidates than lanes
    x[200:300, 1:] = -math.inf
    x[300:400] = -math.inf
    x[400:500, ::3] = math.nan
    x[500:600] += torch.randn((100, 64), device=dev()) * 1e-7
    x[600:700, 5] = math.inf
    b = torch.zeros(64, device=dev()) if bias else None
    check(x, 6, "softmax", b, groups, max(1, groups // 2))
    check(x, 6, "sigmoid", b, groups, max(1, groups // 2))


@pytest.mark.parametrize("tokens", [3, 70])
def test_in_front_of_the_experts(tokens):
    """Router logits -> route_experts -> fused_moe_gguf: the same as with weights and ids formed by torch."""
    e, hidden, inter = 16, 512, 256
    _, w1 = experts_wire(12, e, 2 * inter, hidden, seed=1)
    _, w2 = experts_wire(8, e, hidden, inter, seed=2)
    _, x = act(tokens, hidden, seed=3, dt="bf16")
    x = x * 0.02
    r = logits(tokens, e, "bf16", seed=5)
    w, ids = linear.route_experts(r, 4)
    got = linear.fused_moe_gguf(x, w1, w2, w, ids, 12, 8)
    top, at = torch.sort(r.float().softmax(-1), dim=-1, descending=True, stable=True)
    assert torch.equal(at[:, :4].to(torch.int32), ids)
    want = linear.fused_moe_gguf(x, w1, w2, w, at[:, :4], 12, 8)
    assert torch.equal(got, want) and bool(torch.isfinite(got).all())


def test_refusals():
    x = torch.zeros((4, 64), device=dev())
    f = linear.route_experts
    for bad in (lambda: f(x, 0), lambda: f(x, 65), lambda: f(x, 33), lambda: f(x, 8, groups=3), lambda: f(x, 8, groups=8, top_groups=9), lambda: f(x, 8, groups=0),
                lambda: f(x, 9, groups=8, top_groups=1), lambda: f(x, 2, groups=64, top_groups=4), lambda: f(x, 8, bias=x[0].half()), lambda: f(x, 8, bias=x[0, :8]),
                lambda: f(x.double(), 8), lambda: f(x[0], 8), lambda: f(x.t(), 2), lambda: f(x.long(), 8), lambda: f(torch.zeros((1, 1025), device=dev()), 8),
                lambda: f(x.clone().requires_grad_(), 8), lambda: f(x, 8, bias=torch.zeros(64))):
        with pytest.raises(RuntimeError):
            bad()
    with pytest.raises(ValueError):
        f(x, 8, scoring="top")
