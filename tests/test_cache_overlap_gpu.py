"""Caches that share memory with each other or with the input are refused, caches side by side in one tensor are not."""
import pytest
import torch

from kaillm_b200 import attention
from tests.gpu_util import dev

pytestmark = pytest.mark.gpu

PAGES, PAGE, KV, D = 5, 4, 2, 64


def call(k, v, qkv=None):
    g = torch.Generator().manual_seed(3)
    t = 6
    x = torch.randn((t, 8 * D), generator=g).half().to(dev()) if qkv is None else qkv
    slots = torch.tensor([19, 0, 7, -1, 12, 5], device=dev())
    q = attention.qk_norm_rope_store(x, torch.arange(t, device=dev()), torch.rand(D // 2, generator=g).to(dev()), 4, k, v, slots)
    return q, x, slots


def zeros(*shape):
    return torch.zeros(shape, dtype=torch.float16, device=dev())


def side_by_side():
    """Pairs of views of one tensor that share no element."""
    return {
        "page by page": (lambda c: (c[:, 0], c[:, 1]))(zeros(PAGES, 2, PAGE, KV, D)),
        "token by token": (lambda c: (c[:, :, 0], c[:, :, 1]))(zeros(PAGES, PAGE, 2, KV, D)),
        "heads behind heads": (lambda c: (c[:, :, :KV], c[:, :, KV:]))(zeros(PAGES, PAGE, 2 * KV, D)),
        "heads in turn": (lambda c: (c[:, :, 0::2], c[:, :, 1::2]))(zeros(PAGES, PAGE, 2 * KV, D)),
        "head by head": (lambda c: (c[..., :D], c[..., D:]))(zeros(PAGES, PAGE, KV, 2 * D)),
        "heads first": (lambda c: (c[:, 1].transpose(1, 2), c[:, 0].transpose(1, 2)))(zeros(PAGES, 2, KV, PAGE, D)),
        "one behind the other": (lambda c: (c[:PAGES], c[PAGES:]))(zeros(2 * PAGES, PAGE, KV, D)),
        "pages in turn": (lambda c: (c[0::2], c[1::2]))(zeros(2 * PAGES, PAGE, KV, D)),
    }


@pytest.mark.parametrize("name", ["page by page", "token by token", "heads behind heads", "heads in turn", "head by head", "heads first", "one behind the other",
                                  "pages in turn"])
def test_side_by_side(name):
    k, v = side_by_side()[name]
    want_k, want_v = zeros(PAGES, PAGE, KV, D), zeros(PAGES, PAGE, KV, D)
    want = call(want_k, want_v)[0]
    got, x, slots = call(k, v)
    assert torch.equal(got, want) and torch.equal(k, want_k) and torch.equal(v, want_v)
    for i, s in enumerate(slots.tolist()):
        assert s < 0 or torch.equal(v[s // PAGE, s % PAGE].flatten(), x[i, 6 * D:])


def test_overlaps_are_refused():
    c = zeros(PAGES + 1, PAGE, KV, D)
    wide = zeros(PAGES, 3, PAGE, KV, D)
    heads = zeros(PAGES, PAGE, KV + 1, D)
    pairs = [(c, c), (c[:-1], c[1:]), (c[1:], c[:-1]), (wide[:, 0], wide[:, 0]), (heads[:, :, :-1], heads[:, :, 1:]),
             (c.flatten()[:-64].view(-1)[:PAGES * PAGE * KV * D].view(PAGES, PAGE, KV, D), c.flatten()[8:8 + PAGES * PAGE * KV * D].view(PAGES, PAGE, KV, D))]
    for k, v in pairs:
        with pytest.raises(RuntimeError, match="overlap"):
            call(k, v)
    flat = zeros(6 * 8 * D)
    k = flat[:PAGES * PAGE * KV * D].view(PAGES, PAGE, KV, D)
    for k, v in ((k, c[:-1]), (c[:-1], k)):
        with pytest.raises(RuntimeError, match="qkv"):
            call(k, v, flat.view(6, 8 * D))
