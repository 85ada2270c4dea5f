"""The operators' calls past the dispatcher: the same results, and whoever watches operators still sees them."""
import threading

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from kaillm_b200 import attention, linear, ops
from tests.gpu_util import dev

pytestmark = pytest.mark.gpu


def calls():
    g = torch.Generator().manual_seed(0)
    qkv = torch.randn((5, 8 * 64), generator=g).to(torch.bfloat16).to(dev())
    pos = torch.arange(5, device=dev())
    freq = torch.rand(32, generator=g).to(dev())
    k, v = (torch.randn((4, 16, 2, 64), generator=g).to(torch.bfloat16).to(dev()) for _ in range(2))
    slots = torch.tensor([3, 17, -1, 40, 63], device=dev())
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev())    # noqa: E731
    q = torch.randn((2, 4, 64), generator=g).to(torch.bfloat16).to(dev())
    x = torch.randn((7, 24), generator=g).to(dev())
    return {
        "qk_norm_rope": (qkv, pos, freq, 4, 2, None, None, 1e-6, False, 1.0),
        "qk_norm_rope_store": (qkv, pos, freq, 4, k, v, slots, None, torch.ones(64, dtype=torch.bfloat16, device=dev()), 1e-6, True, 1.5),
        "paged_attention": (q, k, v, i32([0, 1], [2, 3]), i32(20, 32), 0.125, 0, 0.0, True),
        "plan_pages": (i32([0, -1], [2, 3]), i32(16, 20), i32(3, 4), i32(1), i32(0), 16, 9),
        "moe_route": (x, 3, True, torch.rand(24, generator=g).to(dev()), 4, 2, True, 2.0),
    }


def flat(r):
    return [r] if isinstance(r, torch.Tensor) else list(r)


NAMES = ["qk_norm_rope", "qk_norm_rope_store", "paged_attention", "plan_pages", "moe_route"]


@pytest.mark.parametrize("name", NAMES)
def test_the_same_as_the_overload(name):
    here, there = calls()[name], calls()[name]
    direct, overload = getattr(ops, name.upper()), getattr(torch.ops._C_gguf, name).default
    got, want = flat(direct(*here)), flat(overload(*there))
    assert len(got) == len(want) and all(type(a) is torch.Tensor and a.dtype == b.dtype and a.shape == b.shape for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip(here, there) if isinstance(a, torch.Tensor))      # tables and caches written in place
    with torch.inference_mode():
        assert all(torch.equal(a, b) for a, b in zip(flat(direct(*here)), flat(overload(*there))))
    with pytest.raises((RuntimeError, TypeError)):
        direct(*here[:-1])
    with pytest.raises((RuntimeError, TypeError)):
        direct(*here[:-1], "text")
    with pytest.raises(RuntimeError):
        direct(here[0].cpu(), *here[1:])


@pytest.mark.parametrize("name", NAMES)
def test_modes_see_the_operator(name):
    seen = []

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    args = calls()[name]
    with Watch():
        getattr(ops, name.upper())(*args)
    assert f"_C_gguf.{name}.default" in seen

    class Functions(torch.overrides.TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            seen.append("function " + str(func))
            return func(*args, **(kwargs or {}))

    with Functions():
        getattr(ops, name.upper())(*args)
    assert any(s.startswith("function") and name in s for s in seen)
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
        getattr(ops, name.upper())(*args)
    assert any(e.key == f"_C_gguf::{name}" for e in prof.key_averages())


def test_other_types_of_arguments():
    x = calls()["moe_route"][0]
    want = linear.route_experts(x, 3, scale=2.0)
    for k, scale in ((torch.tensor(3), 2.0), (3, 2), (True + 2, 2.0)):
        got = linear.route_experts(x, int(k), scale=scale)
        assert all(torch.equal(a, b) for a, b in zip(got, want))

    class Sub(torch.Tensor):
        pass

    got = linear.route_experts(x.as_subclass(Sub), 3, scale=2.0)
    assert all(torch.equal(a.as_subclass(torch.Tensor), b) for a, b in zip(got, want))
    negative = torch._neg_view(x)
    assert all(torch.equal(a, b) for a, b in zip(linear.route_experts(negative, 3), linear.route_experts(-x, 3)))
    q, k, v, table, lens = calls()["paged_attention"][:5]
    assert torch.equal(attention.paged_attention(torch.nn.Parameter(q, requires_grad=False), k, v, table, lens), attention.paged_attention(q, k, v, table, lens))
    with pytest.raises(RuntimeError, match="derivative"):
        attention.paged_attention(torch.nn.Parameter(q), k, v, table, lens)


def test_threads():
    """Calls from several threads on streams of their own."""
    x = calls()["moe_route"][0]
    want = linear.route_experts(x, 3)
    wrong = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(200):
                got = linear.route_experts(x, 3)
            torch.cuda.current_stream().synchronize()
            if not all(torch.equal(a, b) for a, b in zip(got, want)):
                wrong.append(1)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
