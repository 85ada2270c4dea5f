"""Attention of one token over a paged cache against a 64-bit softmax, at the lengths, layouts and masks where it can go wrong."""
import math

import pytest
import torch

from kaillm_b200 import attention, capi
from tests.attention_util import DT, attend, check_attention, paged_cache
from tests.gpu_util import dev

pytestmark = pytest.mark.gpu


def run(lens, heads, kv, dim, page, dtype, window=0, cap=0.0, seed=0, scale=None, **cache):
    k, v, table = paged_cache(lens, kv, dim, page, dtype, dev(), seed, **cache)
    q = (torch.randn((len(lens), heads, dim), generator=torch.Generator().manual_seed(seed + 1)) * 2).to(DT[dtype]).to(dev())
    n = torch.tensor(lens, dtype=torch.int32, device=dev())
    scale = dim ** -0.5 if scale is None else scale
    got, lse = attention.paged_attention(q, k, v, table, n, scale=scale, window=window, softcap=cap, return_lse=True)
    want, norm, eo, el = attend(q, k, v, table, lens, scale, window, cap)
    check_attention(got, want, eo, dtype)
    empty = torch.isinf(norm)
    assert torch.equal(torch.isinf(lse.cpu()), empty)
    assert bool(((lse.cpu().double() - norm).abs()[~empty] <= el[~empty]).all())
    return q, k, v, table, n, got


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("lens", [[1], [0], [2, 0, 1], [15, 16, 17], [31, 64, 63, 65], [255, 256], [257, 1], [700, 3, 0, 1025, 128]])
def test_lengths(dtype, lens):
    run(lens, 8, 2, 64, 16, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads,kv", [(1, 1), (5, 5), (6, 2), (40, 8), (9, 1), (16, 1), (17, 1), (28, 4), (71, 1), (64, 2)])
def test_head_layouts(dtype, heads, kv):
    run([333, 40], heads, kv, 64, 16, dtype, seed=heads)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 96, 112, 128, 144, 160, 192, 208, 240, 256])
def test_head_dims(dtype, dim):
    run([5, 290], 6, 2, dim, 16, dtype, seed=dim)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("page", [1, 3, 7, 8, 16, 24, 48, 100, 256])
@pytest.mark.parametrize("window", [0, 45])
def test_page_sizes(dtype, page, window):
    run([301, 99, 1, 128], 4, 2, 64, page, dtype, window=window, seed=page)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("window", [1, 2, 16, 17, 100, 999, 1000, 5000])
def test_windows(dtype, window):
    run([1000, 17, 0, 16, 100], 10, 2, 128, 16, dtype, window=window, seed=window)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("cap", [0.5, 20.0])
def test_capped_scores(dtype, cap):
    run([400, 33], 8, 2, 64, 32, dtype, cap=cap)
    run([400, 33], 8, 2, 64, 32, dtype, cap=cap, window=50, scale=2.0)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_long_and_short_together(dtype):
    run([9000, 1, 0, 37, 4096, 2], 8, 1, 128, 16, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_lengths_up_to_the_last_one(dtype):
    """Lengths that a tile more would take past 2^31; the sequences' pages are the same few over and over."""
    page, g = 1 << 20, torch.Generator().manual_seed(5)
    k, v = (torch.randn((2, page, 1, 16), generator=g).to(DT[dtype]).to(dev()) for _ in range(2))
    table = (torch.arange(2 * 2049, dtype=torch.int32, device=dev()) % 2).view(2, 2049)
    lens = [2 ** 31 - 1, 2 ** 31 - 20]
    q = torch.randn((2, 2, 16), generator=g).to(DT[dtype]).to(dev())
    got = attention.paged_attention(q, k, v, table, torch.tensor(lens, dtype=torch.int32, device=dev()), window=300)
    want, _, eo, _ = attend(q, k, v, table, lens, 0.25, 300, 0.0)
    check_attention(got, want, eo, dtype)


@pytest.mark.parametrize("heads,kv,dim", [(8, 8, 128), (20, 2, 64), (16, 1, 256), (18, 9, 96)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_items_enough_for_every_warp(heads, kv, dim, dtype):
    """Many items: warps work on their own; few of them cross from one to the next, one of them over many."""
    lens = [(37 * i) % 211 for i in range(120 if kv < 4 else 40)]
    run(lens, heads, kv, dim, 16, dtype, width=14)                # lengths that need no division
    lens[5] = 2500
    run(lens, heads, kv, dim, 16, dtype)
    run(lens, heads, kv, dim, 8, dtype, window=70)


@pytest.mark.parametrize("heads,kv", [(1, 1), (4, 1), (10, 2), (8, 1), (12, 1)])
@pytest.mark.parametrize("dim", [32, 64, 128, 144, 256])
def test_f32_tiles(heads, kv, dim):
    """Every tile of the fp32 form, at lengths that end inside one, whole and divided."""
    run([5, 0, 190, 64, 1], heads, kv, dim, 16, "f32", seed=dim)
    run([1203, 7, 0, 402], heads, kv, dim, 24, "f32", seed=dim)
    run([1203, 7, 0, 402], heads, kv, dim, 16, "f32", window=333, cap=9.0, seed=dim)


def test_many_sequences():
    """More sequences than one scan step of a CTA covers, in an order of lengths that a static split would serve badly."""
    lens = [(i * i) % 97 for i in range(700)]
    run(lens, 4, 2, 64, 16, "bf16")
    lens[3] = 6000
    run(lens, 4, 2, 64, 16, "bf16")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_head_major_cache_and_strided_queries(dtype):
    q, k, v, table, n, got = run([120, 900], 8, 4, 64, 32, dtype, heads_first=True)
    wide = torch.zeros((2, 8 * 64 + 3 + 512), dtype=DT[dtype], device=dev())
    wide[:, 3:3 + 512] = q.reshape(2, 512)
    same = attention.paged_attention(wide[:, 3:3 + 512].unflatten(1, (8, 64)), k, v, table, n)
    assert torch.equal(same, got)
    swapped = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(attention.paged_attention(swapped, k.contiguous(), v.contiguous(), table, n), got)
    table_wide = torch.full((2, table.shape[1] + 7), -5, dtype=torch.int32, device=dev())
    table_wide[:, 7:] = table
    assert torch.equal(attention.paged_attention(q, k, v, table_wide[:, 7:], n), got)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_strides_that_no_step_follows(dtype):
    """Dimensions of one entry may carry any stride."""
    q, k, v, table, n, got = run([30], 2, 1, 64, 32, dtype, spare=0)
    assert k.shape == (1, 32, 1, 64)
    odd = [c.as_strided(c.shape, (7, 64, 3, 1)) for c in (k, v)]
    assert torch.equal(attention.paged_attention(q.as_strided(q.shape, (5, 64, 1)), *odd, table, n, scale=0.125), got)
    k1, v1 = (c[:1, :1].contiguous().as_strided((1, 1, 1, 64), (3, 5, 7, 1)) for c in (k, v))
    want = attention.paged_attention(q, k[:, :1].contiguous(), v[:, :1].contiguous(), table, torch.ones_like(n))
    assert torch.equal(attention.paged_attention(q, k1, v1, table, torch.ones_like(n)), want)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_absent_pages_and_lengths_beyond_the_table(dtype):
    lens = [200, 64, 500]
    k, v, table = paged_cache(lens, 2, 64, 16, dtype, dev(), spare=2)
    table[0, 3], table[0, 12], table[1, :4], table[2, 5] = -1, 2 ** 31 - 1, -7, k.shape[0]
    q = torch.randn((3, 4, 64), device=dev()).to(DT[dtype])
    asked = [200, 64, 100000]                       # the table of sequence 2 ends at 512 tokens, of which 500 are filled
    last = int(table[2, 31])
    k[last, 4:], v[last, 4:] = 0.25, 0.5
    got = attention.paged_attention(q, k, v, table, torch.tensor(asked, dtype=torch.int32, device=dev()), scale=0.125)
    want, _, eo, _ = attend(q, k, v, table, asked, 0.125, 0, 0.0)
    check_attention(got, want, eo, dtype)
    assert bool((got[1] == 0).all())
    none = attention.paged_attention(q, k, v, table[:, :0], torch.tensor([5, -3, 0], dtype=torch.int32, device=dev()))
    assert bool((none == 0).all())


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_extreme_scores(dtype):
    """One key far above all others: its value comes out; keys of equal scores: their mean."""
    k, v, table = paged_cache([600], 1, 64, 16, dtype, dev())
    q = torch.zeros((1, 2, 64), dtype=DT[dtype], device=dev())
    q[0, 0, 0] = 100.0
    name, place = int(table[0, 437 // 16]), 437 % 16
    k[..., 0] = k[..., 0].clamp(-5, 5)
    k[name, place, 0, 0] = 300.0
    got = attention.paged_attention(q, k, v, table, torch.tensor([600], dtype=torch.int32, device=dev()), scale=1.0)
    assert torch.equal(got[0, 0], v[name, place, 0])
    want, _, eo, _ = attend(q, k, v, table, [600], 1.0, 0, 0.0)
    check_attention(got[:, 1:], want[:, 1:], eo[:, 1:], dtype)


def test_repeated_calls_agree_and_leave_the_inputs():
    q, k, v, table, n, got = run([5000, 77, 2500], 40, 8, 128, 16, "bf16")
    before = [t.clone() for t in (q, k.nan_to_num(7), v.nan_to_num(7), table, n)]
    for _ in range(5):
        assert torch.equal(attention.paged_attention(q, k, v, table, n), got)
    assert all(torch.equal(a, b) for a, b in zip(before, (q, k.nan_to_num(7), v.nan_to_num(7), table, n)))


def test_captured_calls_follow_the_lengths():
    """Two graphs over one cache, replayed on two streams at once with lengths that change between replays."""
    lens = [3000, 1200, 64]
    k, v, table = paged_cache(lens, 2, 128, 16, "bf16", dev())
    q = torch.randn((3, 10, 128), device=dev()).to(torch.bfloat16)
    n = [torch.tensor(lens, dtype=torch.int32, device=dev()) for _ in range(2)]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    attention.paged_attention(q, k, v, table, n[0])
    torch.cuda.synchronize()
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            outs.append(attention.paged_attention(q * (i + 1), k, v, table, n[i]))
    for now in ([3000, 1200, 64], [1, 0, 33], [2999, 5, 0]):
        for i in range(2):
            n[i].copy_(torch.tensor(now if i == 0 else now[::-1], dtype=torch.int32).clamp_max(64 if i else 3000))
        torch.cuda.synchronize()
        for _ in range(8):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], attention.paged_attention(q * (i + 1), k, v, table, n[i]))


def test_side_stream():
    lens = [2000, 10]
    k, v, table = paged_cache(lens, 2, 64, 16, "f16", dev())
    n = torch.tensor(lens, dtype=torch.int32, device=dev())
    q = torch.randn((2, 4, 64), device=dev()).to(torch.float16)
    want = attention.paged_attention(q, k, v, table, n)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        late = torch.zeros_like(q)
        for _ in range(20):
            late = late * 0 + q                    # produced on the side stream
        got = attention.paged_attention(late, k, v, table, n)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_cache_beyond_32_bit_offsets(dtype):
    """Pages whose first element lies behind 2^32, written by the rotation and read back."""
    kv, d, page, n = 8, 128, 16, 75
    pages = 2 ** 32 // (page * kv * d) + 40
    kc, vc = (torch.empty((pages, page, kv, d), dtype=DT[dtype], device=dev()) for _ in range(2))
    table = torch.tensor([[pages - 1, pages - 30, 3, pages - 2, pages - 17]], dtype=torch.int32, device=dev())
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn((n, (16 + 2 * kv) * d), generator=g).to(DT[dtype]).to(dev())
    at = torch.arange(n, device=dev())
    slots = table[0].long()[at // page] * page + at % page
    freq = torch.rand(d // 2, generator=g).to(dev())
    q = attention.qk_norm_rope_store(qkv, at, freq, 16, kc, vc, slots)
    _, k = attention.qk_norm_rope(qkv, at, freq, 16, kv)
    assert torch.equal(kc[table[0].long()].flatten(0, 1)[:n], k) and torch.equal(vc[table[0].long()].flatten(0, 1)[:n], qkv[:, 24 * d:].unflatten(1, (kv, d)))
    lens = torch.tensor([n], dtype=torch.int32, device=dev())
    got = attention.paged_attention(q[-1:], kc, vc, table, lens, scale=0.1)
    few = table[0].long()
    small = torch.arange(5, dtype=torch.int32, device=dev())[None]
    want, _, eo, _ = attend(q[-1:], kc[few], vc[few], small, [n], 0.1, 0, 0.0)
    check_attention(got, want, eo, dtype)
    wide = torch.cat([table, torch.full((1, 60), -1, dtype=torch.int32, device=dev())], 1)      # divided among workers
    check_attention(attention.paged_attention(q[-1:], kc, vc, wide, lens, scale=0.1), want, eo, dtype)


def test_two_graphs_at_once():
    """Captured calls with scratch of their own, replayed on two streams at the same time."""
    sets = []
    for seed, lens in ((1, [3000, 7, 900, 1500]), (2, [1, 4000, 2500, 0, 333])):
        k, v, table = paged_cache(lens, 4, 128, 16, "bf16", dev(), seed)
        q = torch.randn((len(lens), 16, 128), generator=torch.Generator().manual_seed(seed)).bfloat16().to(dev())
        n = torch.tensor(lens, dtype=torch.int32, device=dev())
        want = attention.paged_attention(q, k, v, table, n)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = [attention.paged_attention(q, k, v, table, n) for _ in range(3)]
        sets.append((graph, outs, want, torch.cuda.Stream(), (q, k, v, table, n)))
    for _ in range(20):
        for graph, outs, want, stream, _ in sets:
            with torch.cuda.stream(stream):
                for o in outs:
                    o.zero_()
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for _, outs, want, _, _ in sets for o in outs)


def test_no_wait_has_run_out():
    run([5000, 0, 77], 8, 2, 128, 16, "bf16")
    assert capi.paged_attention_status() == 0


def test_refusals():
    k, v, table = paged_cache([40, 8], 2, 64, 16, "bf16", dev())
    n = torch.tensor([40, 8], dtype=torch.int32, device=dev())
    q = torch.zeros((2, 4, 64), dtype=torch.bfloat16, device=dev())
    f = attention.paged_attention
    assert f(q[:0], k, v, table[:0], n[:0]).shape == (0, 4, 64)
    for bad in (lambda: f(q.half(), k, v, table, n), lambda: f(q, k, v.half(), table, n), lambda: f(q[:, :3], k, v, table, n),
                lambda: f(q[..., :48], k, v, table, n), lambda: f(q, k[..., :40], v[..., :40], table, n),
                lambda: f(q[..., :40], k[..., :40], v[..., :40], table, n), lambda: f(q, k, v[:, :8], table, n),
                lambda: f(q, k, v, table.long(), n), lambda: f(q, k, v, table, n.long()), lambda: f(q, k, v, table[:1], n),
                lambda: f(q, k, v, table, n[:1]), lambda: f(q, k, v, table, n.cpu()), lambda: f(q, k, v, table.t().contiguous().t(), n),
                lambda: f(q, k, v, table, n, window=-1), lambda: f(q, k, v, table, n, softcap=-1.0), lambda: f(q, k, v, table, n, scale=math.nan),
                lambda: f(q, k, v, table, n, scale=0.0), lambda: f(q.double(), k.double(), v.double(), table, n),
                lambda: f(q.clone().requires_grad_(), k, v, table, n), lambda: f(q, k.as_strided((3, 16, 2, 64), (2049, 128, 64, 1)), v[:3], table, n),
                lambda: f(q[0], k, v, table, n)):
        with pytest.raises(RuntimeError):
            bad()
    with torch.no_grad():
        assert f(q.clone().requires_grad_(), k, v, table, n).shape == q.shape
