"""The operators between the projections through `ops` and through the C binding: what `attention` and `linear` return."""
import pytest
import torch

from kaillm_b200 import attention, capi, linear, ops
from tests.gpu_util import dev
from tests.test_direct_calls_gpu import NAMES, calls, flat

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", NAMES)
def test_ops(name):
    here, there = calls()[name], calls()[name]
    got, want = flat(getattr(ops, name)(*here)), flat(getattr(torch.ops._C_gguf, name)(*there))
    assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip(here, there) if isinstance(a, torch.Tensor))


def test_names_of_the_arguments():
    """Every argument of the public functions lands where its name says."""
    qkv, pos, freq, h, kv, *_ = calls()["qk_norm_rope"]
    w = torch.rand(64, device=dev())
    want = ops.qk_norm_rope(qkv, pos, freq, h, kv, w, None, 0.5, True, 2.0)
    got = attention.qk_norm_rope(qkv, pos, freq, h, kv, q_weight=w, eps=0.5, interleaved=True, factor=2.0)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    q, k, v, table, lens, *_ = calls()["paged_attention"]
    want = ops.paged_attention(q, k, v, table, lens, 0.3, 9, 4.0, True)
    assert all(torch.equal(a, b) for a, b in zip(attention.paged_attention(q, k, v, table, lens, scale=0.3, window=9, softcap=4.0, return_lse=True), want))
    assert ops.paged_attention(q, k, v, table, lens, 0.3, 9, 4.0, False)[1] is None
    x, _, _, bias, *_ = calls()["moe_route"]
    want = ops.moe_route(x, 2, True, bias, 6, 3, False, 0.5)
    got = linear.route_experts(x, 2, scoring="sigmoid", bias=bias, groups=6, top_groups=3, renormalize=False, scale=0.5)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("weights", [(False, False), (True, False), (False, True), (True, True)])
def test_c_binding_of_the_rotation(weights):
    qkv, pos, freq, h, kv, *_ = calls()["qk_norm_rope"]
    qw, kw = (torch.rand(64, device=dev()) + 0.5 if w else None for w in weights)
    q, k = qkv.new_empty((5, h, 64)), qkv.new_empty((5, kv, 64))
    capi.qk_norm_rope(qkv, pos, freq, h, kv, q, k, q_weight=qw, k_weight=kw, eps=0.1, interleaved=True, factor=1.5)
    want = attention.qk_norm_rope(qkv, pos, freq, h, kv, q_weight=qw, k_weight=kw, eps=0.1, interleaved=True, factor=1.5)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    _, _, _, _, kc, vc, slots, *_ = calls()["qk_norm_rope_store"]
    kc2, vc2 = kc.clone(), vc.clone()
    capi.qk_norm_rope(qkv, pos, freq, h, kv, q, kc, q_weight=qw, k_weight=kw, v_cache=vc, slots=slots)
    assert torch.equal(q, attention.qk_norm_rope_store(qkv, pos, freq, h, kc2, vc2, slots, q_weight=qw, k_weight=kw))
    assert torch.equal(kc, kc2) and torch.equal(vc, vc2)


def test_c_binding_of_the_attention():
    q, k, v, table, lens, *_ = calls()["paged_attention"]
    out, lse = torch.empty_like(q), torch.empty((2, 4), device=dev())
    scratch = torch.empty(capi.paged_attention_workspace_bytes(2, 4, 2, 64), dtype=torch.uint8, device=dev())
    capi.paged_attention(q, k, v, table, lens, out, scratch, scale=0.2, window=11, softcap=3.0, lse=lse)
    want = attention.paged_attention(q, k, v, table, lens, scale=0.2, window=11, softcap=3.0, return_lse=True)
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    with pytest.raises(capi.KqError, match="scratch"):
        capi.paged_attention(q, k, v, table, lens, out, scratch[:256], scale=0.2)
    assert capi.paged_attention_status() == capi.paged_attention_status(device=dev()) == capi.paged_attention_status(True) == 0
