"""Steps of a stack with attention that run out of pages."""
import pytest
import torch

from kaillm_b200 import sharded
from tests.gpu_util import dev
from tests.test_decode_step_gpu import HIDDEN, M, PAGE, WIDTH, state, weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("case", ["row", "list"])
def test_a_stack_reports_tokens_without_a_page(case, captured):
    lens = [WIDTH * PAGE - 1, 3, 20] if case == "row" else [15, 16, 40]
    att = state(lens)
    if case == "list":
        att.taken.fill_(att.free_pages.numel() - 1)     # one page left: for sequence 1 at once, for sequence 0 a step later none
    stack = sharded.DecoderStack(weights(), M, HIDDEN, dev(), unsharded=True, attention=att)
    h = (torch.randn((M, HIDDEN), device=dev()) * 0.1).to(torch.bfloat16)
    step = lambda: stack.forward(h)    # noqa: E731
    step()
    stack.check()
    if captured:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            stack.forward(h)
        step = graph.replay
    step()
    for _ in range(2):
        with pytest.raises(RuntimeError, match=r"sequences \[0\]"):
            stack.check()
        step()
    assert att.seq_lens.tolist() == [n + 4 for n in lens]
