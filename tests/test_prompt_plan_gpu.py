"""Making a plan beside queued work, and letting go of it before it was read."""

import pytest
import torch

from tests.test_serving_attention_gpu import randn
from xpu_playground_b200 import kernels as K

pytestmark = pytest.mark.gpu
LENS = [300, 17, 500]


def operands():
    return [randn(i, sum(LENS), h, 64) for i, h in enumerate((4, 2, 2))]


def test_making_a_plan_does_not_wait_for_queued_work():
    K.PromptPlan(LENS, 4, 2, 64)
    torch.cuda.synchronize()
    torch.cuda._sleep(400_000_000)  # about 0.2 s
    plan = K.PromptPlan(LENS, 4, 2, 64)
    assert not torch.cuda.current_stream().query()
    out = K.prompt_attention(plan, *operands())[0]
    torch.cuda.synchronize()
    assert torch.equal(out, K.prompt_attention(plan, *operands())[0])


@pytest.mark.parametrize("own_stream", [False, True])
def test_a_plan_that_is_dropped_is_kept_for_the_calls_that_read_it(own_stream):
    ops = operands()
    want = K.prompt_attention(K.PromptPlan(LENS, 4, 2, 64), *ops)[0]
    stream = torch.cuda.Stream() if own_stream else torch.cuda.current_stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(20_000_000)
        out = K.prompt_attention(K.PromptPlan(LENS, 4, 2, 64), *ops)[0]
    others = [K.PromptPlan([n], 4, 2, 64) for n in (817, 5, 200, 816)]  # would take its memory
    torch.cuda.synchronize()
    assert torch.equal(out, want) and len(others) == 4


def test_a_captured_call_reads_a_plan_made_before():
    ops, plan = operands(), K.PromptPlan(LENS, 4, 2, 64)
    want = K.prompt_attention(plan, *ops)[0]
    out, lse = torch.empty_like(want), torch.empty(sum(LENS), 4, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.prompt_attention(plan, *ops, out=out, lse=lse)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
