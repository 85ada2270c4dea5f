"""Bad arguments of the operators between a decode step's projections come back as the documented codes, before any GPU work; the
plain forms that their GPU tests use agree with each other."""
import ctypes
import subprocess
import sys

import pytest
import torch

from kaillm_b200 import capi
from tests.attention_util import attend, paged_cache, pages, rotate, route

OK, EINVAL, EUNSUPPORTED, ESCRATCH, ELIMIT = capi.KQ_OK, capi.KQ_EINVAL, capi.KQ_EUNSUPPORTED, capi.KQ_ESCRATCH, capi.KQ_ELIMIT
S3 = ctypes.c_int64 * 3


def _attend(q=0x1000, dt=2, b=2, h=8, kv=2, d=128, sb=1024, sh=128, k=0x2000, ks=(4096, 256, 128), v=0x3000, vs=(4096, 256, 128), pages=9, page=16,
            table=0x4000, ts=4, width=4, lens=0x5000, scale=0.1, window=0, cap=0.0, out=0x6000, lse=None, scratch=0x7000, sbytes=1 << 30):
    return capi.lib.kq_paged_attention(q, dt, b, h, kv, d, sb, sh, k, S3(*ks), v, S3(*vs), pages, page, table, ts, width, lens, scale, window, cap, out, lse,
                                       scratch, sbytes, None)


def test_paged_attention():
    assert _attend(b=0) == OK
    assert _attend(dt=3) == EUNSUPPORTED and _attend(d=40) == EUNSUPPORTED and _attend(d=272) == EUNSUPPORTED and _attend(d=0) == EUNSUPPORTED
    assert "multiple of 16" in capi.lib.kq_last_error().decode()
    for bad in (dict(b=-1), dict(h=0), dict(kv=0), dict(h=7), dict(page=0), dict(pages=-1), dict(width=-1), dict(window=-1), dict(window=1 << 31), dict(scale=0.0),
                dict(scale=float("nan")), dict(scale=float("inf")), dict(cap=-1.0), dict(cap=float("nan")), dict(q=None), dict(out=None), dict(lens=None),
                dict(table=None), dict(k=None), dict(v=None), dict(k=0x2008), dict(v=0x3002), dict(q=0x1001), dict(out=0x6004), dict(ks=(4097, 256, 128)),
                dict(vs=(4096, 256, 4)), dict(ks=(-4096, 256, 128)), dict(out=0x1000), dict(lens=0x5002), dict(table=0x4001), dict(lse=0x8002),
                dict(scale=2e30), dict(cap=2e30)):
        assert _attend(**bad) == EINVAL, bad
        assert "kq_paged_attention" in capi.lib.kq_last_error().decode()
    assert _attend(scratch=None) == ESCRATCH and _attend(scratch=0x7010) == ESCRATCH and _attend(sbytes=1000) == ESCRATCH
    assert _attend(b=1 << 21) == ELIMIT and _attend(page=1 << 31) == ELIMIT and _attend(width=1 << 31) == ELIMIT and _attend(b=1 << 20, h=1 << 12, kv=1) == ELIMIT
    ws = capi.paged_attention_workspace_bytes
    assert ws(1, 8, 2, 0) == 0 and ws(1, 8, 2, 272) == 0 and ws(1, 8, 3, 64) == 0 and ws(-1, 8, 2, 64) == 0
    assert 0 < ws(1, 8, 2, 64) < ws(1, 8, 2, 256) <= ws(1, 40, 2, 256) < ws(1000, 40, 2, 256) < 64 << 20


def _rope(qkv=0x1000, dt=2, t=4, st=1536, h=8, kv=2, d=128, pos=0x2000, p64=0, freq=0x3000, rot=128, inter=0, qw=None, kw=None, wdt=0, q=0x4000, k=0x5000,
          ks=None, v=None, vs=None, slots=None, s64=0, pages=0, page=0):
    return capi.lib.kq_qk_norm_rope(qkv, dt, t, st, h, kv, d, pos, p64, freq, rot, inter, 1.0, qw, kw, wdt, 1e-6, q, k, ks, v, vs, slots, s64, pages, page, None)


def test_qk_norm_rope():
    cache = dict(v=0x6000, ks=S3(4096, 256, 128), vs=S3(4096, 256, 128), slots=0x7000, pages=3, page=16)
    assert _rope(t=0) == OK and _rope(t=0, **cache) == OK
    assert _rope(dt=9) == EUNSUPPORTED and _rope(d=127, st=1 << 20) == EUNSUPPORTED and _rope(d=514, st=1 << 20) == EUNSUPPORTED
    assert _rope(qw=0x8000, wdt=1) == EUNSUPPORTED and "norm weights" in capi.lib.kq_last_error().decode()
    for bad in (dict(t=-1), dict(h=0), dict(kv=0), dict(rot=130), dict(rot=3), dict(rot=-2), dict(st=1535), dict(qkv=None), dict(pos=None), dict(freq=None), dict(q=None),
                dict(k=None), dict(qkv=0x1001), dict(q=0x4001), dict(freq=0x3002), dict(cache, slots=None), dict(cache, ks=None), dict(cache, vs=None),
                dict(cache, pages=0), dict(cache, page=0), dict(cache, v=0x6001), dict(pos=0x2002), dict(pos=0x2004, p64=1), dict(cache, slots=0x7002),
                dict(cache, slots=0x7004, s64=1), dict(qw=0x8001, wdt=2), dict(kw=0x8002, wdt=0)):
        assert _rope(**bad) == EINVAL, bad
    assert _rope(h=1 << 17) == ELIMIT and _rope(**dict(cache, page=1 << 31)) == ELIMIT and _rope(t=1 << 31) == ELIMIT


def _plan(table=0x1000, ts=8, width=8, seen=0x2000, new=0x3000, r=4, free=0x4000, nfree=10, taken=0x5000, page=16, tokens=5, total=0x6000, starts=0x7000,
          pos=0x8000, slots=0x9000, out=0xa000):
    return capi.lib.kq_plan_pages(table, ts, width, seen, new, r, free, nfree, taken, page, tokens, total, starts, pos, slots, out, None)


def test_plan_pages():
    for bad in (dict(page=0), dict(r=-1), dict(width=-1), dict(nfree=-1), dict(tokens=-1), dict(ts=7), dict(table=None), dict(seen=None), dict(new=None),
                dict(free=None), dict(taken=None), dict(total=None), dict(starts=None), dict(pos=None), dict(slots=None), dict(out=None), dict(out=0x5000),
                dict(total=0x2000), dict(total=0x3000), dict(table=0x1002), dict(seen=0x2001), dict(new=0x3002), dict(free=0x4001), dict(taken=0x5002), dict(total=0x6001),
                dict(starts=0x7002), dict(pos=0x8001), dict(slots=0x9004), dict(out=0xa002)):
        assert _plan(**bad) == EINVAL, bad
    assert _plan(r=(1 << 20) + 1) == ELIMIT and _plan(tokens=1 << 31) == ELIMIT and _plan(page=1 << 31) == ELIMIT


def _route(x=0x1000, dt=0, t=4, e=64, st=64, k=8, sig=0, bias=None, g=1, tg=1, ren=1, w=0x2000, ids=0x3000):
    return capi.lib.kq_moe_route(x, dt, t, e, st, k, sig, bias, g, tg, ren, 1.0, w, ids, None)


def test_moe_route():
    assert _route(t=0) == OK and _route(dt=5) == EUNSUPPORTED
    for bad in (dict(t=-1), dict(e=0), dict(k=0), dict(k=65), dict(g=0), dict(g=3), dict(g=4, tg=0), dict(g=4, tg=5), dict(g=16, tg=1), dict(x=None), dict(w=None), dict(ids=None),
                dict(st=63), dict(x=0x1002), dict(bias=0x4001), dict(w=0x2002), dict(ids=0x3001)):
        assert _route(**bad) == EINVAL, bad
    assert _route(e=1025, st=1025) == ELIMIT and _route(k=33) == ELIMIT and _route(g=64, tg=64) == ELIMIT


def test_plain_forms():
    """The loops of the tests against torch on whole tensors."""
    k, v, table = paged_cache([37], 2, 16, 8, "f32", "cpu")
    q = torch.randn(1, 4, 16)
    out, lse, bound, _ = attend(q, k, v, table, [37], 0.25, 0, 0.0)
    slot = [int(table[0, j // 8]) * 8 + j % 8 for j in range(37)]
    kk, vv = (c.reshape(-1, 2, 16)[slot].double().repeat_interleave(2, 1) for c in (k, v))
    s = torch.einsum("hd,nhd->hn", q[0].double(), kk) * 0.25
    assert torch.allclose(out[0], torch.einsum("hn,nhd->hd", s.softmax(1), vv)) and torch.allclose(lse[0], s.logsumexp(1))
    assert 0 < float(bound.max()) < 1e-3
    x = torch.randn(3, 2, 8)
    y, _ = rotate(x, torch.tensor([0, 1, 2]), torch.ones(4), None, 0.0, False, 1.0)
    assert torch.allclose(y[0], x[0].double()) and torch.allclose(y.pow(2).sum(-1), x.double().pow(2).sum(-1))
    w, ids = route(torch.tensor([[0.0, 2.0, 2.0, 1.0]]), 2, "softmax", None, 2, 1, True, 1.0)
    assert ids.tolist() == [[1, 0]] and w.sum() == pytest.approx(1.0)
    t, total, starts, pos, slots, taken = pages([[3, -1]], [7], [3], [9, 4], 1, 8, 4)
    assert (t, total, starts, pos, slots, taken) == ([[3, 4]], [10], [0, 3], [7, 8, 9, 0], [31, 32, 33, -1], 2)


def test_beside_another_library_of_the_same_namespace():
    """Where the reference's operators are registered already, this package uses those, and says that it has no others."""
    code = """
import torch
lib = torch.library.Library("_C_gguf", "DEF")
lib.define("ggml_mul_mat_vec_a8(Tensor W, Tensor X, int type, int row) -> Tensor")
lib.impl("ggml_mul_mat_vec_a8", lambda W, X, type, row: X + row, "CPU")
from kaillm_b200 import attention, linear, ops
assert ops.ggml_mul_mat_vec_a8(torch.zeros(1), torch.zeros(1), 2, 3).item() == 3
try:
    linear.route_experts(torch.zeros(1, 4), 2)
except ImportError as e:
    assert "moe_route" in str(e)
else:
    raise AssertionError
"""
    subprocess.run([sys.executable, "-c", code], check=True, timeout=300)


def test_calls_that_are_not_plain_reach_the_overload():
    from kaillm_b200 import linear, ops

    for bad in (lambda: linear.route_experts(torch.zeros(2, 8), 2), lambda: ops.MOE_ROUTE(1), lambda: ops.PAGED_ATTENTION(), lambda: ops.PLAN_PAGES(*[None] * 7)):
        with pytest.raises((RuntimeError, NotImplementedError, TypeError)):
            bad()


def test_a_stack_refuses_attention_that_does_not_fit():
    from kaillm_b200 import sharded
    from kaillm_b200.attention import StepAttention

    def att(layers=1, seqs=2, heads=4, kv=2, d=16):
        i32 = lambda *s: torch.zeros(s, dtype=torch.int32)    # noqa: E731
        return StepAttention([[torch.zeros(3, 8, kv, d)] * 2] * layers, heads, torch.ones(d // 2), i32(seqs, 2), i32(seqs), i32(3), i32(1))

    w = {name: (torch.zeros((n, k // 32 * 34), dtype=torch.uint8), 8, n, k) for name, (n, k) in
         {"qkv": (128, 64), "o": (64, 64), "gate_up": (128, 64), "down": (64, 64)}.items()}
    make = lambda a: sharded.DecoderStack([w], 2, 64, torch.device("cpu"), attention=a)    # noqa: E731
    assert make(att()).attention is not None and make(None).attention is None
    for bad in (att(layers=2), att(seqs=3), att(heads=8), att(kv=1), att(d=32)):
        with pytest.raises(ValueError):
            make(bad)
    with pytest.raises(ValueError):
        StepAttention([], 4, torch.ones(8), torch.zeros(1, 1), torch.zeros(1), torch.zeros(1), torch.zeros(1))
    with pytest.raises(ValueError):
        StepAttention([[torch.zeros(3, 8, 2, 16)] * 2], 4, torch.ones(8), torch.zeros(1, 1), torch.zeros(1), torch.zeros(1), torch.zeros(1), q_weights=[])
