"""Norms of queries and keys with the rotation, and the write into the cache, against 64 bits."""
import pytest
import torch

from kaillm_b200 import attention
from tests.attention_util import DT, HALF_STEP, TINY, rotate
from tests.gpu_util import dev

pytestmark = pytest.mark.gpu


def inv_freq(rotated, base=1e6):
    return (base ** (-torch.arange(0, rotated, 2, dtype=torch.float64) / max(rotated, 1))).float().to(dev())


def inputs(t, h, kv, d, dtype, norm, seed=0, w_dtype=None, far=100000):
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn((t, (h + 2 * kv) * d), generator=g) * 3).to(DT[dtype]).to(dev())
    pos = torch.randint(0, far, (t,), generator=g).to(torch.int32).to(dev())
    w = [(torch.randn(d, generator=g) * 0.3 + 1).to(DT[w_dtype or dtype]).to(dev()) if norm else None for _ in range(2)]
    return qkv, pos, w


def close(got, want, bound, dtype):
    got = got.double().cpu()
    limit = bound * (1 + HALF_STEP[dtype]) + HALF_STEP[dtype] * want.abs() + TINY[dtype]
    off = (got - want).abs()
    assert bool((off <= limit).all()), float((off / limit).max())


def check(qkv, pos, freq, h, kv, d, w, dtype, eps=1e-6, interleaved=False, factor=1.0):
    x = qkv.cpu().reshape(qkv.shape[0], h + 2 * kv, d)
    q, k = attention.qk_norm_rope(qkv, pos, freq, h, kv, q_weight=w[0], k_weight=w[1], eps=eps, interleaved=interleaved, factor=factor)
    for got, rows, weight in ((q, x[:, :h], w[0]), (k, x[:, h:h + kv], w[1])):
        assert got.dtype == qkv.dtype and got.shape == rows.shape and got.is_contiguous()
        close(got, *rotate(rows, pos, freq, weight, eps, interleaved, factor), dtype)
    return q, k


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("t,h,kv,d", [(1, 40, 8, 128), (3, 1, 1, 64), (17, 6, 2, 256), (300, 5, 5, 80), (9, 7, 1, 2), (5, 3, 3, 34), (4, 2, 1, 512), (2, 71, 1, 96),
                                      (700, 28, 4, 128)])
def test_sizes(dtype, norm, t, h, kv, d):
    qkv, pos, w = inputs(t, h, kv, d, dtype, norm)
    check(qkv, pos, inv_freq(d), h, kv, d, w, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rotated", [(128, 128), (128, 64), (256, 64), (80, 20), (64, 2), (64, 0), (128, 126), (48, 48)])
def test_pairs_and_partial_rotation(dtype, interleaved, d, rotated):
    qkv, pos, w = inputs(13, 4, 2, d, dtype, True, seed=d)
    check(qkv, pos, inv_freq(rotated), 4, 2, d, w, dtype, interleaved=interleaved)
    check(qkv, pos, inv_freq(rotated), 4, 2, d, [None, w[1]], dtype, interleaved=interleaved)


@pytest.mark.parametrize("far", [2 ** 20, 2 ** 31 - 1])
def test_far_positions(far):
    qkv, pos, w = inputs(50, 4, 2, 128, "f32", False, far=far)
    pos[0], pos[1] = far, -5
    check(qkv, pos, inv_freq(128), 4, 2, 128, w, "f32")
    check(qkv, pos.long() * 3, inv_freq(128), 4, 2, 128, w, "f32")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_weights_eps_factor_strides(dtype):
    qkv, pos, w = inputs(21, 4, 2, 128, dtype, True, w_dtype="f32")
    freq = inv_freq(128)
    q, k = check(qkv, pos, freq, 4, 2, 128, w, dtype, eps=0.3, factor=1.37)
    wide = torch.zeros((21, qkv.shape[1] + 5), dtype=qkv.dtype, device=dev())
    wide[:, 1:1 + qkv.shape[1]] = qkv              # rows at odd addresses
    for view in (wide[:, 1:1 + qkv.shape[1]],):
        got = attention.qk_norm_rope(view, pos, freq, 4, 2, q_weight=w[0], k_weight=w[1], eps=0.3, factor=1.37)
        for a, b in zip(got, (q, k)):              # another order of a sum of 128 squares at most
            assert bool(((a.double() - b.double()).abs() <= 2 * HALF_STEP[dtype] * b.double().abs() + 2.0 ** -15).all())
    zero = torch.zeros_like(qkv)
    assert all(bool((t == 0).all()) for t in attention.qk_norm_rope(zero, pos, freq, 4, 2, q_weight=w[0], k_weight=w[1]))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("t,page,d,slot64", [(1, 16, 128, True), (50, 16, 128, True), (50, 7, 80, False), (400, 1, 64, False), (33, 48, 256, True)])
@pytest.mark.parametrize("heads_first", [False, True])
def test_store(dtype, t, page, d, slot64, heads_first):
    h, kv = 6, 2
    qkv, pos, w = inputs(t, h, kv, d, dtype, True, seed=t)
    freq = inv_freq(d)
    pages = -(-t // page) + 3
    shape = (pages, kv, page, d) if heads_first else (pages, page, kv, d)
    kc, vc = (torch.full(shape, 9.0, dtype=DT[dtype], device=dev()) for _ in range(2))
    if heads_first:
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(1))[:t]
    if t > 10:
        slots[3], slots[7], slots[9] = -1, pages * page, -2 ** 31
    idx = slots.to(torch.int64 if slot64 else torch.int32).to(dev())
    q = attention.qk_norm_rope_store(qkv, pos, freq, h, kc, vc, idx, q_weight=w[0], k_weight=w[1])
    q2, k2 = attention.qk_norm_rope(qkv, pos, freq, h, kv, q_weight=w[0], k_weight=w[1])
    assert torch.equal(q, q2)
    close(q, *rotate(qkv.cpu().reshape(t, -1, d)[:, :h], pos, freq, w[0], 1e-6, False, 1.0), dtype)
    want_k, want_v = (torch.full((pages * page, kv, d), 9.0, dtype=DT[dtype], device=dev()) for _ in range(2))
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < pages * page:
            want_k[s], want_v[s] = k2[i], qkv[i].reshape(-1, d)[h + kv:]
    assert torch.equal(kc.reshape(-1, kv, d), want_k) and torch.equal(vc.reshape(-1, kv, d), want_v)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("h,kv,d,rotated,interleaved", [(40, 8, 128, 128, False), (9, 3, 64, 64, True), (5, 2, 256, 64, False), (5, 3, 80, 48, True), (2, 1, 128, 0, False),
                                                        (7, 7, 16, 16, False), (3, 1, 256, 256, True), (6, 2, 96, 96, False), (5, 5, 80, 48, False),
                                                        (5, 2, 80, 40, False), (3, 3, 72, 72, True), (4, 1, 40, 8, False), (2, 2, 256, 24, True)])
def test_many_tokens(dtype, h, kv, d, rotated, interleaved):
    """So many that a warp takes a token."""
    many(dtype, 20 * 160 + 1, h, kv, d, rotated, interleaved)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("t", [12, 700])
@pytest.mark.parametrize("h,kv,d,rotated,interleaved", [(5, 2, 80, 40, False), (71, 1, 80, 40, True), (3, 3, 72, 72, True), (4, 1, 40, 8, False), (2, 2, 256, 24, True),
                                                        (9, 2, 20, 20, False), (3, 1, 128, 128, True)])
def test_small_pieces(dtype, t, h, kv, d, rotated, interleaved):
    many(dtype, t, h, kv, d, rotated, interleaved)


def many(dtype, t, h, kv, d, rotated, interleaved):
    page = 16
    qkv, pos, w = inputs(t, h, kv, d, dtype, True, seed=d)
    qkv[5, d - 1] = float("nan")                   # of the first head of one token
    freq = inv_freq(rotated)
    x = qkv.cpu().reshape(t, h + 2 * kv, d)
    kc, vc = (torch.full((t // page + 3, page, kv, d), 9.0, dtype=DT[dtype], device=dev()) for _ in range(2))
    slots = torch.randperm(kc.shape[0] * page, generator=torch.Generator().manual_seed(1))[:t]
    slots[3], slots[7], slots[9] = -1, kc.shape[0] * page, -2 ** 31
    free = torch.ones(kc.shape[0] * page, dtype=torch.bool)
    rest = torch.ones(t, dtype=torch.bool)
    rest[[3, 7, 9]] = False
    free[slots[rest]] = False
    for weights in (w, [None, w[1]]):
        q = attention.qk_norm_rope_store(qkv, pos, freq, h, kc, vc, slots.to(dev()), q_weight=weights[0], k_weight=weights[1], interleaved=interleaved)
        bad = torch.isnan(q.cpu())
        bad_at = bad.nonzero()[:, :2].unique(dim=0).tolist()
        assert bad_at == [[5, 0]] and (weights[0] is None or bool(bad[5, 0].all()))
        q[5, 0], qkv0 = 0, x[5, 0].clone()
        x[5, 0] = 0
        close(q, *rotate(x[:, :h], pos, freq, weights[0], 1e-6, interleaved, 1.0), dtype)
        x[5, 0] = qkv0
        kept = kc.reshape(-1, kv, d)[slots[rest].to(dev())]
        want, bound = rotate(x[:, h:h + kv], pos, freq, weights[1], 1e-6, interleaved, 1.0)
        close(kept, want[rest], bound[rest] if torch.is_tensor(bound) else bound, dtype)
        assert torch.equal(vc.reshape(-1, kv, d)[slots[rest].to(dev())].cpu(), x[rest, h + kv:])
        assert bool((kc.reshape(-1, kv, d).cpu()[free] == 9.0).all()) and bool((vc.reshape(-1, kv, d).cpu()[free] == 9.0).all())
    dense = attention.qk_norm_rope(qkv, pos, freq, h, kv, q_weight=None, k_weight=w[1], interleaved=interleaved)
    assert torch.equal(dense[1][rest.to(dev())], kept)


def test_nothing_to_do_and_capture():
    qkv, pos, w = inputs(4, 4, 2, 128, "bf16", True)
    freq = inv_freq(128)
    q, k = attention.qk_norm_rope(qkv[:0], pos[:0], freq, 4, 2)
    assert q.shape == (0, 4, 128) and k.shape == (0, 2, 128)
    want = attention.qk_norm_rope(qkv, pos, freq, 4, 2, q_weight=w[0], k_weight=w[1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = attention.qk_norm_rope(qkv, pos, freq, 4, 2, q_weight=w[0], k_weight=w[1])
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    pos.add_(11)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, attention.qk_norm_rope(qkv, pos, freq, 4, 2, q_weight=w[0], k_weight=w[1])))


def test_refusals():
    qkv, pos, w = inputs(4, 4, 2, 64, "bf16", True)
    freq = inv_freq(64)
    cache = torch.zeros((3, 16, 2, 64), dtype=torch.bfloat16, device=dev())
    slots = torch.arange(4, device=dev())
    f, s = attention.qk_norm_rope, attention.qk_norm_rope_store
    for bad in (lambda: f(qkv, pos, freq, 4, 3), lambda: f(qkv[0], pos, freq, 4, 2), lambda: f(qkv.t(), pos, freq, 4, 2), lambda: f(qkv, pos[:3], freq, 4, 2),
                lambda: f(qkv, pos.float(), freq, 4, 2), lambda: f(qkv, pos, freq.double(), 4, 2), lambda: f(qkv, pos, inv_freq(66), 4, 2),
                lambda: f(qkv, pos, freq, 4, 2, q_weight=w[0].half()), lambda: f(qkv, pos, freq, 4, 2, q_weight=w[0][:32]),
                lambda: f(qkv, pos, freq, 4, 2, q_weight=w[0], k_weight=w[1].float()), lambda: f(qkv.double(), pos, freq, 4, 2), lambda: f(qkv, pos.cpu(), freq, 4, 2),
                lambda: f(qkv, pos, freq, 0, 2), lambda: f(qkv.clone().requires_grad_(), pos, freq, 4, 2),
                lambda: f(qkv, pos, freq, 4, 2, k_weight=w[1].clone().requires_grad_()),
                lambda: s(qkv, pos, freq, 4, cache.half(), cache, slots), lambda: s(qkv, pos, freq, 4, cache, cache[:, :8], slots),
                lambda: s(qkv, pos, freq, 4, cache[..., :32], cache[..., :32], slots), lambda: s(qkv, pos, freq, 4, cache, cache.clone(), slots[:3]),
                lambda: s(qkv, pos, freq, 4, cache, cache.clone(), slots.float()), lambda: s(qkv, pos, freq, 4, cache[:0], cache[:0], slots),
                lambda: s(qkv, pos, freq, 4, cache[:1].expand(3, 16, 2, 64), cache, slots)):
        with pytest.raises(RuntimeError):
            bad()
