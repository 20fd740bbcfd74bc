"""Sampling where places are counted and where blocks' counters are joined, against a sort in 64 bits."""

import pytest
import torch

from tests.test_sample_gpu import BF16, FP16, INF, NAN, check, randn, settings
from xpu_playground_b200 import kernels as K

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 20, 40, 90])  # eight, four, two and one block a row
@pytest.mark.parametrize("vocabulary", [31, 32, 33, 64, 65, 127, 128, 129, 255, 256, 257, 300])
def test_as_many_tokens_as_places(rows, vocabulary):
    """All are listed where top-k is 256: a multiple of a warp or not, to the last place."""
    g = torch.Generator().manual_seed(vocabulary)
    u = torch.rand(rows, generator=g)
    u[-1] = 1 - 2.0 ** -24
    x = randn(rows, rows, vocabulary, FP16)
    check(x, u, top_k=[256] * rows)
    check(x[:, :1].expand(rows, vocabulary).contiguous(), u, top_k=[min(256, i + vocabulary // 2) for i in range(rows)])
    check(x, u, top_k=[1 + 3 * i % 256 for i in range(rows)], top_p=[0.9] * rows, temperature=[3.0] * rows)


@pytest.mark.parametrize("rows", [1, 8, 20, 40])
@pytest.mark.parametrize("many", [60000, 65535, 65536, 80000, 131072])
def test_a_value_that_blocks_share(rows, many):
    """Groups whose joined counter holds the value's number, and one whose does not, beside one another."""
    vocabulary = 151936
    g = torch.Generator().manual_seed(many + rows)
    x = randn(many, rows, vocabulary, BF16)
    for row in x:
        places = torch.randperm(vocabulary, generator=g)
        row[places[:many]] = 4.0
        row[places[many:many + 2000]] = 4.03125  # its neighbour, in the same group
        row[places[many + 2000:many + 5000]] = 5.0
        row[places[many + 5000:many + 5300]] = -0.0
        row[places[many + 5300:many + 5600]] = 0.0
    u = torch.rand(rows, generator=g)
    u[0] = 0.999
    check(x, u)
    check(x, u, temperature=[0.8] * rows, top_p=[0.7] * rows, min_p=[0.05] * rows)
    check(x, u, top_k=[1000 + 997 * i for i in range(rows)])
    check(x, u, temperature=[20.0] * rows, min_p=[0.75] * rows)
    check(x, u, temperature=[50.0] * rows, top_k=[140000] * rows)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("vocabulary", [1, 2, 63, 100, 511, 513, 1024, 2047, 2048, 2049])
def test_short_rows(vocabulary, dtype):
    """On both sides of the length up to which a row is sorted whole: any settings, ties, masks and rows without an answer."""
    rows = 300
    x = randn(vocabulary, rows, vocabulary, dtype)
    x[:40] = (2 * x[:40]).round() / 2  # ties, zeros of both signs
    x[40:60, 1::2] = -INF
    x[60:70, : vocabulary - 1] = torch.finfo(dtype).min
    x[70:74] = -INF
    x[74:76, vocabulary // 2] = INF
    x[76:78, vocabulary - 1] = NAN
    x[78:80, 0] = -torch.tensor(NAN)
    u = torch.rand(rows, generator=torch.Generator().manual_seed(vocabulary))
    u[::50], u[1::50] = 0.0, 1 - 2.0 ** -24
    tokens, _ = check(x, u, **settings(vocabulary, rows))
    assert (tokens[70:80] == -1).all()
    check(x, u)
    apart = torch.empty(rows, vocabulary + 3, dtype=dtype, device="cuda")[:, 1:vocabulary + 1]  # rows at odd places
    apart.copy_(x)
    check(apart, u, **settings(vocabulary + 1, rows))


@pytest.mark.parametrize("vocabulary", [1000, 5000])
def test_captured_with_other_numbers(vocabulary):
    x, u = randn(3, 64, vocabulary, BF16).cuda(), torch.rand(64, device="cuda")
    tokens, logprobs = torch.empty(64, dtype=torch.int32, device="cuda"), torch.empty(64, device="cuda")
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        K.sample(x, u, tokens=tokens, logprobs=logprobs)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        K.sample(x, u, tokens=tokens, logprobs=logprobs)
    for seed in range(3):
        u.copy_(torch.rand(64, generator=torch.Generator().manual_seed(seed)))
        x.copy_(randn(seed, 64, vocabulary, BF16))
        graph.replay()
        want = check(x, u.cpu())
        assert torch.equal(tokens, want[0]) and torch.equal(logprobs, want[1])
