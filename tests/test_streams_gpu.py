"""Calls on another stream than the current one, outputs allocated by the call."""

import pytest
import torch

from tests.test_serving_attention_gpu import BF16, as_int64, make_cache, randn
from xpu_playground_b200 import kernels as K

pytestmark = pytest.mark.gpu
N = 1024  # outputs of 1024 rows of 8 x 128: a block that the allocator would hand out again


def prompt():
    q, k, v = (randn(i, N, h, 128) for i, h in enumerate((8, 2, 2)))
    plan = K.PromptPlan([N], 8, 2, 128)
    return lambda stream=None: K.prompt_attention(plan, q, k, v, stream=stream)[0]


def tree():
    cache, _ = make_cache([100] * 16, 2, 128, 16, BF16, 5)
    q, k, v = (randn(i, N, h, 128) for i, h in enumerate((8, 2, 2)))
    ids = torch.arange(16, dtype=torch.int32, device="cuda")
    starts = torch.arange(0, N + 1, 64, dtype=torch.int32, device="cuda")
    sets, ws = as_int64([(1 << (i % 64 + 1)) - 1 for i in range(N)]), K.tree_attention_workspace(16, N, 8, 2, 128)
    return lambda stream=None: K.tree_attention(cache, 1, ids, starts, sets, q, k, v, ws, stream=stream)[0]


def gemm_bt():
    a, w = randn(1, N, 256), randn(2, 1024, 256)
    return lambda stream=None: K.gemm_bt(a, w, stream=stream)


def gemv():
    a, x = randn(1, N * 1024, 64), randn(2, 64)
    return lambda stream=None: K.gemv(a, x, stream=stream)


@pytest.mark.parametrize("make", [prompt, tree, gemm_bt, gemv])
def test_outputs_do_not_take_memory_that_the_current_stream_still_reads(make):
    call = make()
    want = call()
    held = torch.full_like(want, 7.0)
    side, out = torch.cuda.Stream(), None
    side.wait_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    torch.cuda._sleep(20_000_000)  # about 10 ms
    copy = held.clone()            # queued behind it
    del held                       # free for the current stream's next allocation, and for no other's
    out = call(side)
    torch.cuda.synchronize()
    assert bool((copy == 7.0).all()) and torch.equal(out, want)


@pytest.mark.parametrize("make", [prompt, tree, gemm_bt, gemv])
def test_results_that_are_dropped_are_not_handed_out_under_a_reader(make):
    call = make()
    want = call()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    out = call(side)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda._sleep(20_000_000)
    copy = out.clone()  # on the current stream, later
    del out
    with torch.cuda.stream(side):
        others = [torch.full_like(want, 3.0) for _ in range(4)]
    torch.cuda.synchronize()
    assert torch.equal(copy, want) and len(others) == 4
