"""Page tables and slots from request lengths against the same rules in Python."""
import pytest
import torch

from kaillm_b200 import attention
from tests.attention_util import pages
from tests.gpu_util import dev

pytestmark = pytest.mark.gpu


def run(seen, new, page, width, free, taken=0, pad=0, table=None):
    n = len(seen)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev())    # noqa: E731
    table = [[1000 * r + j for j in range(width)] for r in range(n)] if table is None else table
    tokens = sum(max(v, 0) for v in new) + pad
    want = pages(table, seen, new, free, taken, page, tokens)
    t = i32(table).reshape(n, width)
    got = attention.plan_pages(t, i32(seen), i32(new), i32(free), i32([taken]), page, tokens)
    for a, b in zip((t, *got[:4]), want[:5]):
        assert a.tolist() == b
    assert got[4].tolist() == [want[5]]
    assert got[3].dtype == torch.int64 and all(a.dtype == torch.int32 for a in (*got[:3], got[4]))
    return t, got


@pytest.mark.parametrize("page", [1, 3, 16, 100])
@pytest.mark.parametrize("seen,new", [([0], [1]), ([0, 0], [0, 0]), ([5], [40]), ([16, 15, 17, 0], [1, 1, 1, 1]), ([7, 0, 48, 31], [0, 33, 16, 2]),
                                      ([100, 3], [0, 0]), ([-4, 2], [3, -9])])
def test_small(page, seen, new):
    run(seen, new, page, 160, list(range(50000, 50400)), taken=2, pad=3)


@pytest.mark.parametrize("requests,seed", [(31, 0), (1023, 1), (1024, 2), (1025, 3), (2500, 4)])
def test_many_requests(requests, seed):
    g = torch.Generator().manual_seed(seed)
    seen = torch.randint(0, 70, (requests,), generator=g).tolist()
    new = torch.randint(0, 20, (requests,), generator=g).tolist()
    free = (torch.randperm(2 * requests + 9, generator=g) + 10 ** 7).tolist()
    run(seen, new, 16, 8, free, taken=5, pad=1)


def test_long_prompts_over_several_ctas():
    run([0, 3, 4096], [30000, 0, 9999], 16, 3000, list(range(100000, 104000)), pad=777)


def test_the_list_runs_out_and_rows_end():
    t, got = run([0, 10, 0], [64, 30, 20], 16, 4, list(range(70, 75)), taken=1)
    assert int(got[4]) > 5 and (t == -1).any() and (got[3] == -1).any()
    run([60, 0], [30, 5], 16, 4, list(range(70, 90)))          # 90 tokens in a row of 64
    run([200], [3], 16, 4, [1, 2, 3])                          # already beyond the row
    run([0, 0], [5, 5], 16, 2, [])
    run([3], [2], 16, 0, [5], table=[[]])
    run([], [], 16, 4, [1, 2], pad=4, table=[])


def test_num_tokens_below_the_sum_writes_nothing_behind_it():
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev())    # noqa: E731
    table = torch.full((2, 4), -9, dtype=torch.int32, device=dev())
    total, starts, positions, slots, taken = attention.plan_pages(table, i32([0, 0]), i32([20, 20]), i32([7, 8, 9, 10]), i32([0]), 16, 18)
    assert positions.tolist() == list(range(18)) and slots.tolist() == [112 + i for i in range(16)] + [128, 129]
    assert table.tolist() == [[7, 8, -9, -9], [-9] * 4] and taken.tolist() == [4] and starts.tolist() == [0, 20, 40]


def test_steps_in_a_captured_loop():
    """A decode loop as a graph: lengths, table and cursor move on from replay to replay."""
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev())    # noqa: E731
    seen, new, free, cursor = i32([15, 0, 30]), i32([1, 1, 1]), i32(list(range(40, 60))), i32([0])
    table = torch.full((3, 4), -1, dtype=torch.int32, device=dev())
    table[0, 0], table[2, 0], table[2, 1] = 1, 2, 3
    state = (table.tolist(), seen.tolist(), 0)
    warm = [t.clone() for t in (table, seen, cursor)]
    attention.plan_pages(warm[0], warm[1], new, free, warm[2], 16, 4)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        total, starts, positions, slots, after = attention.plan_pages(table, seen, new, free, cursor, 16, 4)
        seen.copy_(total)
        cursor.copy_(after)
    for _ in range(20):
        graph.replay()
        t, n, st, pos, sl, took = pages(state[0], state[1], [1, 1, 1], free.tolist(), state[2], 16, 4)
        assert table.tolist() == t and seen.tolist() == n and positions.tolist() == pos and slots.tolist() == sl and cursor.tolist() == [took]
        state = (t, n, took)


def test_refusals():
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev())    # noqa: E731
    t, a, f, c = torch.zeros((2, 4), dtype=torch.int32, device=dev()), i32([1, 2]), i32([3, 4]), i32([0])
    p = attention.plan_pages
    for bad in (lambda: p(t.long(), a, a, f, c, 16, 4), lambda: p(t, a.long(), a, f, c, 16, 4), lambda: p(t, a, a[:1], f, c, 16, 4),
                lambda: p(t, a, a, f.cpu(), c, 16, 4), lambda: p(t, a, a, f, a, 16, 4), lambda: p(t, a, a, f, c, 0, 4), lambda: p(t, a, a, f, c, 16, -1),
                lambda: p(t.t(), a, a, f, c, 16, 4), lambda: p(t[:1].expand(2, 4), a, a, f, c, 16, 4)):
        with pytest.raises(RuntimeError):
            bad()
