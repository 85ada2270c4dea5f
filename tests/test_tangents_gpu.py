"""Forward-mode differentiation: the operators have no derivative and refuse inputs that carry a tangent."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from kaillm_b200 import ops
from tests.gpu_util import dev
from tests.test_direct_calls_gpu import calls

pytestmark = pytest.mark.gpu

FLOATS = [("qk_norm_rope", 0), ("qk_norm_rope", 2), ("qk_norm_rope_store", 0), ("qk_norm_rope_store", 4), ("qk_norm_rope_store", 5), ("qk_norm_rope_store", 8),
          ("paged_attention", 0), ("paged_attention", 1), ("paged_attention", 2), ("moe_route", 0), ("moe_route", 3)]


@pytest.mark.parametrize("name,at", FLOATS)
def test_tangents_are_refused(name, at):
    args = list(calls()[name])
    plain = args[at]
    for call in (getattr(ops, name.upper()), getattr(torch.ops._C_gguf, name).default):
        with fwd.dual_level():
            args[at] = fwd.make_dual(plain, torch.ones_like(plain))
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="derivative"):
                    call(*args)
            with fwd._set_fwd_grad_enabled(False):
                call(*args)
        args[at] = plain
        call(*args)


@pytest.mark.parametrize("name,at", FLOATS)
@pytest.mark.parametrize("transform", ["grad", "jvp", "vjp", "jacfwd"])
def test_transforms_are_refused(name, at, transform):
    args = list(calls()[name])
    plain = args[at]

    def f(x):
        out = getattr(ops, name.upper())(*args[:at], x, *args[at + 1:])
        return (out if isinstance(out, torch.Tensor) else out[0]).sum()

    run = {"grad": lambda: torch.func.grad(f)(plain), "jvp": lambda: torch.func.jvp(f, (plain,), (torch.ones_like(plain),)),
           "vjp": lambda: torch.func.vjp(f, plain), "jacfwd": lambda: torch.func.jacfwd(f)(plain)}[transform]
    with pytest.raises(RuntimeError, match="derivative"):
        run()


def test_inputs_that_nobody_differentiates_pass_through_a_transform():
    q, k, v, table, lens, *rest = calls()["paged_attention"]
    want = ops.PAGED_ATTENTION(q, k, v, table, lens, *rest)[0]
    got = torch.func.grad(lambda x: (x * ops.PAGED_ATTENTION(q, k, v, table, lens, *rest)[0].float()).sum())(torch.ones(want.shape, device=dev()))
    assert torch.equal(got, want.float())
    both = torch.func.vmap(lambda x: ops.PAGED_ATTENTION(x, k, v, table, lens, *rest)[0])(torch.stack([q, q * 2]))
    assert torch.equal(both[0], want)
    with torch.no_grad():
        assert torch.equal(torch.ops._C_gguf.paged_attention(q.clone().requires_grad_(), k, v, table, lens, *rest)[0], want)
