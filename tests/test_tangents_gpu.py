"""Forward-mode differentiation: the operators have no derivative and refuse inputs that carry a tangent."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from kaillm_b200 import ops
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
