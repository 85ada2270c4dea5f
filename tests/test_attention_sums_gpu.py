"""Long sums of the 16-bit attention kernels: no drift with the number of keys."""
import pytest
import torch

from kaillm_b200 import attention
from tests.attention_util import attend, paged_cache
from tests.gpu_util import dev

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("group,dim,times", [(8, 64, 2048), (12, 64, 2048), (5, 256, 1024)])
def test_long_sums_do_not_drift(group, dim, times):
    """The same 512 keys `times` times over (the table names their pages again and again) give what they give once, up to the rounding of
    the output, whose errors have no direction: values in [1, 2), outputs near 1.5 and off by at most 2^-11 each, evenly spread, so
    the mean over n of them has the deviation 2^-10 / sqrt(12) / 1.5 / sqrt(n), of which five are allowed.  Besides, with
    u = 2^-24: a weight kept as two fp16 parts is off by 2^-22 at most, and rounded sums have no direction either; 2^-19 for all of
    that.  A running sum that the products cut off instead of rounding loses half a step each time: single outputs came out up to 1.5
    steps too small here."""
    batch, kv, n = 9, 4, 512
    k, v, table = paged_cache([n], kv, dim, 64, "f16", dev(), spare=0)
    g = torch.Generator().manual_seed(2)
    v.copy_((torch.rand(v.shape, generator=g) + 1).half())
    q = torch.randn((batch, kv * group, dim), generator=g).half().to(dev())
    wide = table.repeat(batch, times)
    lens = torch.full((batch,), n * times, dtype=torch.int32, device=dev())
    got = attention.paged_attention(q, k, v, wide, lens).double().cpu()
    want, _, _, _ = attend(q, k, v, table.repeat(batch, 1), [n] * batch, dim ** -0.5, 0, 0.0)
    off = (got - want) / want
    assert float(off.abs().max()) < 2.0 ** -11
    bound = 5 * 2.0 ** -10 / 12 ** 0.5 / 1.5 / got.numel() ** 0.5 + 2.0 ** -19
    assert abs(float(off.mean())) < bound, (float(off.mean()), bound)
