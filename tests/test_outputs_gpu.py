"""Every output of an operator is a tensor of its own."""
import pytest
import torch
from torch._subclasses.schema_check_mode import SchemaCheckMode

from kaillm_b200 import ops
from tests.test_direct_calls_gpu import NAMES, calls, flat

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", NAMES)
def test_outputs_share_no_memory(name):
    for call in (getattr(ops, name.upper()), getattr(torch.ops._C_gguf, name).default):
        got = flat(call(*calls()[name]))
        assert len({t.untyped_storage().data_ptr() for t in got}) == len(got)
        assert all(t.untyped_storage().nbytes() == t.numel() * t.element_size() and t.storage_offset() == 0 for t in got)
        for i, t in enumerate(got):                     # grows over nobody
            others = [(o, o.clone()) for j, o in enumerate(got) if j > i]
            t.resize_(t.numel() + 64).fill_(77)
            assert all(torch.equal(o, c) for o, c in others)


@pytest.mark.parametrize("name", NAMES)
def test_schemas_hold(name):
    with SchemaCheckMode():                             # aliases and writes that a schema does not declare raise
        getattr(ops, name.upper())(*calls()[name])
