"""What a decode step's attention reports and refuses, without a GPU."""
import pytest
import torch

from kaillm_b200 import capi, sharded
from kaillm_b200.attention import StepAttention


def step_attention(layers=1, seqs=2, heads=4, kv=2, d=16, width=2):
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)    # noqa: E731
    return StepAttention([[torch.zeros(3, 8, kv, d), torch.zeros(3, 8, kv, d)] for _ in range(layers)], heads, torch.ones(d // 2), i32(seqs, width), i32(seqs), i32(3), i32(1))


def layer(qkv=128, o=64):
    return {name: (torch.zeros((n, k // 32 * 34), dtype=torch.uint8), 8, n, k) for name, (n, k) in
            {"qkv": (qkv, 64), "o": (64, o), "gate_up": (128, 64), "down": (64, 64)}.items()}


def test_a_stack_reports_an_attention_that_gave_up(monkeypatch):
    status = {"value": 0}
    monkeypatch.setattr(capi, "read_status", lambda *a: 0)
    monkeypatch.setattr(capi, "paged_attention_status", lambda clear=False, device=None: status["value"])
    stack = sharded.DecoderStack([layer()], 2, 64, torch.device("cpu"), attention=step_attention())
    plain = sharded.DecoderStack([layer()], 2, 64, torch.device("cpu"))
    stack.check()
    status["value"] = 1
    plain.check()
    with pytest.raises(RuntimeError, match="paged attention"):
        stack.check()


@pytest.mark.parametrize("free,width", [([5, 6], 2), ([5, 6, 7, 8, 9, 4], 1)])
def test_a_token_without_a_page_is_reported(monkeypatch, free, width):
    """The list runs out for the second sequence; the row of both ends."""
    from kaillm_b200 import attention
    from tests.attention_util import pages

    def plan(table, seen, new, free_pages, taken, page, tokens):
        t, *rest, after = pages(table.tolist(), seen.tolist(), new.tolist(), free_pages.tolist(), int(taken), page, tokens)
        table.copy_(torch.tensor(t, dtype=torch.int32))
        total, starts, positions, slots = (torch.tensor(v) for v in rest)
        return total.int(), starts.int(), positions.int(), slots, torch.tensor([after], dtype=torch.int32)

    monkeypatch.setattr(attention, "plan_pages", plan)
    monkeypatch.setattr(capi, "paged_attention_status", lambda clear=False, device=None: 0)
    att = step_attention(width=width)
    att.free_pages = torch.tensor(free, dtype=torch.int32)
    for _ in range(8):                       # the first page of each
        att.begin_step()
    att.check()
    if width == 2:                           # one more page, for one of them
        att.free_pages = torch.tensor(free + [7], dtype=torch.int32)
    att.begin_step()
    lost = [1] if width == 2 else [0, 1]
    for _ in range(2):                       # and it stays so
        with pytest.raises(RuntimeError, match=str(lost).replace("[", r"\[")):
            att.check()
        att.begin_step()
    att.dropped.zero_()
    att.check()


def test_qk_norm_rope_refuses_outputs_that_are_inputs_or_each_other():
    from tests.test_decode_ops_cpu import EINVAL, S3, _rope

    cache = dict(v=0x6000, ks=S3(4096, 256, 128), vs=S3(4096, 256, 128), slots=0x7000, pages=3, page=16)
    for bad in (dict(q=0x1000), dict(k=0x1000), dict(q=0x5000), dict(cache, v=0x5000), dict(cache, v=0x1000), dict(cache, v=0x4000)):
        assert _rope(**bad) == EINVAL, bad
        assert "outputs" in capi.lib.kq_last_error().decode()


def test_a_stack_checks_the_projections_of_every_layer():
    make = lambda *layers: sharded.DecoderStack(list(layers), 2, 64, torch.device("cpu"), attention=step_attention(layers=len(layers)))    # noqa: E731
    assert make(layer(), layer()).attention is not None
    for bad in ((layer(), layer(qkv=160)), (layer(), layer(), layer(o=96))):
        with pytest.raises(ValueError, match="projections"):
            make(*bad)


def test_c_entries_refuse_outputs_that_are_inputs_or_each_other():
    from tests.test_decode_ops_cpu import EINVAL, _attend, _plan, _route

    ins, outs = {"table": 0x1000, "seen": 0x2000, "new": 0x3000, "free": 0x4000, "taken": 0x5000}, ["total", "starts", "pos", "slots", "out"]
    bad = [(_plan, {o: at}) for o in outs for at in ins.values()] + [(_plan, {a: 0xb000, b: 0xb000}) for a in outs for b in outs if a != b]
    bad += [(_plan, {"table": at}) for name, at in ins.items() if name != "table"]
    bad += [(_route, dict(w=0x1000)), (_route, dict(ids=0x1000)), (_route, dict(w=0x3000)), (_route, dict(bias=0x2000)), (_route, dict(bias=0x3000))]
    bad += [(_attend, dict(out=0x2000)), (_attend, dict(out=0x3000)), (_attend, dict(lse=0x6000))]
    for call, args in bad:
        assert call(**args) == EINVAL, (call, args)
        message = capi.lib.kq_last_error().decode()
        assert "must be neither" in message or "must not be another input" in message, (args, message)


def test_attention_made_in_inference_mode_steps_outside(monkeypatch):
    from kaillm_b200 import attention

    with torch.inference_mode():
        att = step_attention()
    att.seq_lens, att.taken = att.seq_lens.clone(), att.taken.clone()
    monkeypatch.setattr(attention, "plan_pages", lambda *a: (att.seq_lens + 1, None, att.seq_lens, torch.tensor([3, -1]), att.taken))
    att.begin_step()
    assert att.dropped.tolist() == [0, -1]
