"""Keys and values that are not finite, visible ones and those that nobody sees."""
import math

import pytest
import torch

from kaillm_b200 import attention
from tests.attention_util import DT, attend, check_attention, paged_cache
from tests.gpu_util import dev

pytestmark = pytest.mark.gpu


def inputs(lens, dtype, heads=6, kv=2, dim=64, page=16):
    k, v, table = paged_cache(lens, kv, dim, page, dtype, dev(), seed=4)
    q = torch.randn((len(lens), heads, dim), generator=torch.Generator().manual_seed(5)).to(DT[dtype]).to(dev())
    return q, k, v, table, torch.tensor(lens, dtype=torch.int32, device=dev())


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n", [40, 2500])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_a_visible_value_spoils_its_column_alone(dtype, n, bad):
    q, k, v, table, lens = inputs([n, 70], dtype)
    at = n // 2
    v[int(table[0, at // 16]), at % 16, 1, 7] = bad                   # of key head 1: query heads 3, 4, 5
    got = attention.paged_attention(q, k, v, table, lens)
    spoiled = torch.zeros(got.shape, dtype=torch.bool)
    spoiled[0, 3:, 7] = True
    assert torch.equal(~torch.isfinite(got.cpu()), spoiled)
    clean = v.clone()
    clean[int(table[0, at // 16]), at % 16, 1, 7] = 0
    want, _, eo, _ = attend(q, k, clean, table, [n, 70], 0.125, 0, 0.0)
    got[spoiled.to(dev())] = 0
    want[spoiled], eo[spoiled] = 0, 0
    check_attention(got, want, eo, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n", [40, 2500])
def test_scores_of_infinity(dtype, n):
    """A key at infinity: heads that score it -infinity go on without it, heads that score it +infinity give no numbers (0 / 0), as in
    the formula; other key heads and sequences do not notice."""
    q, k, v, table, lens = inputs([n, 70], dtype)
    at = n - 3
    q[0, 3, 9], q[0, 4, 9], q[0, 5, 9] = -1.0, 2.0, -0.5
    k[int(table[0, at // 16]), at % 16, 1, 9] = math.inf
    got, lse = attention.paged_attention(q, k, v, table, lens, return_lse=True)
    assert bool(torch.isnan(got[0, 4]).all()) and bool(torch.isnan(lse[0, 4]))
    k[int(table[0, at // 16]), at % 16, 1, 9] = 0
    want, _, eo, _ = attend(q, k, v, table, [n, 70], 0.125, 0, 0.0)      # heads 3 and 5: again below, without that key
    slots = [int(table[0, j // 16]) * 16 + j % 16 for j in range(n)]
    keys, values = (c.cpu().flatten(0, 1)[slots, 1].double() for c in (k, v))
    for h in (3, 5):
        s = keys @ q[0, h].cpu().double() * 0.125
        s[at] = -math.inf
        want[0, h] = torch.softmax(s, 0) @ values
    got[0, 4], want[0, 4], eo[0, 4] = 0, 0, 0
    check_attention(got, want, eo, dtype)
    assert bool(torch.isfinite(lse[0, [0, 1, 2, 3, 5]]).all()) and bool(torch.isfinite(lse[1]).all())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("bad", [math.inf, -math.inf])
def test_infinities_that_nobody_sees(dtype, bad):
    """Behind the length, in front of the window, in pages of nobody: no trace."""
    lens = [333, 18]
    q, k, v, table, n = inputs(lens, dtype)
    want = attention.paged_attention(q, k, v, table, n, window=100)
    seen = torch.zeros(k.shape[:2], dtype=torch.bool)
    for b, length in enumerate(lens):
        for j in range(max(0, length - 100), length):
            seen[int(table[b, j // 16]), j % 16] = True
    k[~seen.to(dev())], v[~seen.to(dev())] = bad, bad
    assert torch.equal(attention.paged_attention(q, k, v, table, n, window=100), want) and bool(torch.isfinite(want).all())
