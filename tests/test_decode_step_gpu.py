"""A decode step of a stack with attention: page tables, cache writes and attention between the projections, step after step."""
import pytest
import torch

from kaillm_b200 import sharded, synth
from kaillm_b200.attention import StepAttention, paged_attention, plan_pages, qk_norm_rope, qk_norm_rope_store
from tests.attention_util import attend, check_attention, rotate
from tests.gpu_util import dev
from tests.test_rope_gpu import close, inv_freq

pytestmark = pytest.mark.gpu

LAYERS, M, HEADS, KV, D, PAGE, WIDTH = 2, 3, 8, 2, 64, 16, 6
HIDDEN, FFN = HEADS * D, 512


def weights():
    out = []
    for layer in range(LAYERS):
        shapes = {"qkv": (8, (HEADS + 2 * KV) * D, HIDDEN), "o": (8, HIDDEN, HIDDEN), "gate_up": (12, 2 * FFN, HIDDEN), "down": (14, HIDDEN, FFN)}
        out.append({name: (torch.from_numpy(synth.wire_numpy(t, n, k, seed=10 * layer + i)).to(dev()), t, n, k) for i, (name, (t, n, k)) in enumerate(shapes.items())})
    return out


def state(lens, norm=True):
    """Caches with random tokens for `lens`, pages handed out in turn."""
    g = torch.Generator(device=dev()).manual_seed(7)
    pages = M * WIDTH + 2
    caches = [tuple(torch.randn((pages, PAGE, KV, D), generator=g, device=dev()).to(torch.bfloat16) for _ in range(2)) for _ in range(LAYERS)]
    table, at = torch.full((M, WIDTH), -1, dtype=torch.int32), 0
    for b, n in enumerate(lens):
        for i in range(-(-n // PAGE)):
            table[b, i] = at
            at += 1
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev())    # noqa: E731
    w = [[(torch.rand(D, generator=g, device=dev()) + 0.5).to(torch.bfloat16) for _ in range(LAYERS)] for _ in range(2)] if norm else (None, None)
    return StepAttention(caches, HEADS, inv_freq(D), table.to(dev()), i32(lens), i32(list(range(at, pages))), i32([0]), q_weights=w[0], k_weights=w[1])


def copy_of(att):
    c = lambda t: t.clone()    # noqa: E731
    return StepAttention([(c(k), c(v)) for k, v in att.caches], HEADS, att.inv_freq, c(att.block_table), c(att.seq_lens), att.free_pages, c(att.taken),
                         q_weights=att.q_weights, k_weights=att.k_weights)


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip([*sum(a.caches, ()), a.block_table, a.seq_lens, a.taken], [*sum(b.caches, ()), b.block_table, b.seq_lens, b.taken]))


def test_steps_against_their_parts_and_64_bits():
    att = state([15, 0, 40])
    stack = sharded.DecoderStack(weights(), M, HIDDEN, dev(), unsharded=True, attention=att)
    h = (torch.randn((M, HIDDEN), device=dev()) * 0.1).to(torch.bfloat16)
    lens = [15, 0, 40]
    for step in range(3):
        before = copy_of(att)
        seen = {}
        stack.forward(h, on_output=lambda li, name, out, prep: seen.__setitem__((li, name), out.clone()))
        lens = [n + 1 for n in lens]
        assert att.seq_lens.tolist() == lens
        # the parts, called one by one on the state before
        total, _, pos, slots, taken = plan_pages(before.block_table, before.seq_lens, torch.ones_like(before.seq_lens), before.free_pages, before.taken, PAGE, M)
        assert total.tolist() == lens and torch.equal(before.block_table, att.block_table) and torch.equal(taken, att.taken) and pos.tolist() == [n - 1 for n in lens]
        for li in range(LAYERS):
            qkv, (kc, vc) = seen[li, "qkv"], before.caches[li]
            q = qk_norm_rope_store(qkv, pos, att.inv_freq, HEADS, kc, vc, slots, q_weight=att.q_weights[li], k_weight=att.k_weights[li])
            out = paged_attention(q, kc, vc, before.block_table, total)
            assert torch.equal(kc, att.caches[li][0]) and torch.equal(vc, att.caches[li][1])
            # and against 64 bits: the new keys in the cache, the attention over what the cache holds
            x = qkv.cpu().reshape(M, HEADS + 2 * KV, D)
            k_new = torch.stack([kc[int(s) // PAGE, int(s) % PAGE] for s in slots])
            close(k_new, *rotate(x[:, HEADS:HEADS + KV], pos, att.inv_freq, att.k_weights[li], 1e-6, False, 1.0), "bf16")
            want, _, eo, _ = attend(q, kc, vc, before.block_table, lens, D ** -0.5, 0, 0.0)
            check_attention(out, want, eo, "bf16")
            # the o projection read exactly this
            probe = sharded.DecoderStack(weights(), M, HIDDEN, dev(), unsharded=True)
            w, t, n, k = probe.w[li]["o"]
            probe._capi.prepare_q8(out.flatten(1), t, n, probe.scratch)
            assert torch.equal(probe._project("o", w, t, n, k), seen[li, "o"])
        h = seen[LAYERS - 1, "down"].clamp(-1, 1)


def test_captured_steps_equal_eager_ones():
    att = state([31, 16, 5], norm=False)
    other = copy_of(att)
    w = weights()
    h = (torch.randn((M, HIDDEN), device=dev()) * 0.1).to(torch.bfloat16)
    eager = sharded.DecoderStack(w, M, HIDDEN, dev(), unsharded=True, attention=att)
    graphed = sharded.DecoderStack(w, M, HIDDEN, dev(), unsharded=True, attention=other)
    start = copy_of(other)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graphed.forward(h)                          # once outside the capture
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip([*sum(other.caches, ()), other.block_table, other.seq_lens, other.taken],
                    [*sum(start.caches, ()), start.block_table, start.seq_lens, start.taken]):
        a.copy_(b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = graphed.forward(h)
    for _ in range(40):
        want = eager.forward(h).clone()
        graph.replay()
        assert torch.equal(out, want) and same(att, other)
    eager.check()
    graphed.check()


def test_prompt_through_qk_norm_rope_and_slots():
    """A prompt's keys stored in one call, then read token by token: the same as keys stored step by step."""
    t = 37
    qkv = torch.randn((t, (HEADS + 2 * KV) * D), device=dev()).to(torch.bfloat16)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev())    # noqa: E731
    caches = [[torch.zeros((4, PAGE, KV, D), dtype=torch.bfloat16, device=dev()) for _ in range(2)] for _ in range(2)]
    tables = [torch.full((1, 4), -1, dtype=torch.int32, device=dev()) for _ in range(2)]
    free = i32([2, 0, 3, 1])
    total, _, pos, slots, _ = plan_pages(tables[0], i32([0]), i32([t]), free, i32([0]), PAGE, t)
    qk_norm_rope_store(qkv, pos, inv_freq(D), HEADS, *caches[0], slots)
    seen, taken = i32([0]), i32([0])
    for i in range(t):
        seen, _, p, s, taken = plan_pages(tables[1], seen, i32([1]), free, taken, PAGE, 1)
        q = qk_norm_rope_store(qkv[i:i + 1], p, inv_freq(D), HEADS, *caches[1], s)
    assert torch.equal(tables[0], tables[1]) and all(torch.equal(a, b) for a, b in zip(*caches))
    whole = qk_norm_rope(qkv, pos, inv_freq(D), HEADS, KV)[0]
    assert torch.equal(whole[-1:], q)
    out = paged_attention(q, *caches[0], tables[0], total)
    want, _, eo, _ = attend(q, *caches[0], tables[0], [t], D ** -0.5, 0, 0.0)
    check_attention(out, want, eo, "bf16")
