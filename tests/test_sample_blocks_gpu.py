"""Sampling of rows too long to be sorted whole, by one, two, four and eight blocks a row, against a sort in 64 bits: rows and
settings that are not numbers, zeros, odd addresses, lists of every size, counters that overflow."""

import re

import pytest
import torch

from tests._graphs import kernels_of
from tests.test_sample_gpu import BF16, FP16, INF, NAN, check, randn, settings
from xpu_playground_b200 import kernels as K

pytestmark = pytest.mark.gpu

# vocabulary, rows, blocks a row: the most with which all rows are resident at once, and no fewer than 4096 logits a block
LENGTHS = [(2500, 12, 1), (9999, 160, 1), (9999, 12, 2), (20000, 12, 4), (40000, 12, 8), (151936, 12, 8), (151936, 24, 4)]


def blocks(logits):
    """Blocks a row of the kernel that is launched; 0: the one for short rows."""
    logits, u = logits.cuda(), torch.zeros(len(logits), device="cuda")
    names = kernels_of(lambda: K.sample(logits, u))
    assert len(names) == 1
    if "k_sample_short" in names[0]:
        return 0
    return int(re.search(r"k_sampleI\w+?Li(\d)E", names[0])[1])


def in_turn(values, rows):
    return [values[i % len(values)] for i in range(rows)]


@pytest.mark.parametrize("vocabulary,rows,size", [(1000, 12, 0), (2048, 12, 0), (2049, 12, 1), *LENGTHS])
def test_blocks_a_row(vocabulary, rows, size):
    assert blocks(torch.zeros(rows, vocabulary, dtype=BF16)) == size and blocks(torch.zeros(rows, vocabulary, dtype=FP16)) == size


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("vocabulary,rows,size", LENGTHS)
def test_rows_that_are_not_numbers(vocabulary, rows, size, dtype):
    """A NaN or an infinity in the first, the last and every other block's run; next to nothing; nothing."""
    x = randn(5, rows, vocabulary, dtype)
    negative_nan = torch.tensor([-1], dtype=torch.int16).view(dtype)
    places = [0, 1, vocabulary // 16, vocabulary // 8 + 3, vocabulary // 4 + 1, vocabulary // 2, 3 * vocabulary // 4, vocabulary - 1]
    for i, place in enumerate(places):
        x[i, place] = [torch.tensor(NAN, dtype=dtype), torch.tensor(INF, dtype=dtype), negative_nan[0]][i % 3]
    x[8] = -INF
    x[9, 3:] = -INF
    x[10, :vocabulary - 1] = -INF
    x[rows - 1, vocabulary // 3] = -INF
    bad = list(range(9))
    for top_k in ([0], [1], [40], [1000], [0, 1, 40, 1000]):
        tokens, _ = check(x, in_turn([0.5, 0.0, 0.999], rows), top_k=in_turn(top_k, rows))
        assert (tokens[bad] == -1).all() and (tokens[9:] >= 0).all()
    tokens, _ = check(x, [0.5] * rows, temperature=[0.0] * rows)
    assert (tokens[bad] == -1).all()


@pytest.mark.parametrize("vocabulary,rows,size", LENGTHS)
def test_settings_that_are_not_numbers(vocabulary, rows, size):
    x = randn(6, rows, vocabulary, BF16)
    for top_k in (0, 40):
        check(x, in_turn([0.1, -0.1, 1.0, NAN, INF, 0.5, 0.5, 0.5, 0.5, 0.5, 0.5, 0.5], rows),
              temperature=in_turn([1, 1, 1, 1, 1, NAN, -1.0, 1, 1, 1, INF, 1e-40], rows),
              top_k=in_turn([top_k] * 7 + [-1] + [top_k] * 4, rows), top_p=in_turn([1] * 8 + [NAN, 1, 1, 1], rows),
              min_p=in_turn([0] * 9 + [NAN, 0, 0], rows))
        # beyond their range: as if at its end
        check(x, in_turn([0.3, 0.9], rows), top_k=[top_k] * rows, top_p=in_turn([-1.0, 0.0, 2.0, -INF, INF], rows),
              min_p=in_turn([-1.0, 5.0, 1.0, 0.0, INF, -INF, 1.5], rows))


@pytest.mark.parametrize("vocabulary,rows,size", LENGTHS)
def test_zeros_of_both_signs_are_equal(vocabulary, rows, size):
    x = torch.zeros(rows, vocabulary, dtype=BF16)
    x[:, ::3] = -0.0
    u = (torch.arange(rows) / rows).float()
    check(x, u, top_k=in_turn([0, 1, 2, 500, 2000], rows))
    check(x.half(), u, temperature=in_turn([0.0, 1.0], rows))
    x[:, 1::3] = -torch.finfo(BF16).tiny * 2.0 ** -7  # the value next to zero
    check(x, u, top_p=in_turn([1.0, 0.5, 0.9], rows))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("shift", range(1, 8))
@pytest.mark.parametrize("vocabulary,rows,size", [(5000, 9, 1), (9999, 9, 2), (20001, 5, 4), (40007, 5, 8)])
def test_rows_at_any_address(vocabulary, rows, size, shift, dtype):
    held = torch.full((rows, vocabulary + 13), INF, dtype=dtype, device="cuda")  # never looked at
    x = held[:, shift:shift + vocabulary]
    x.copy_(randn(9, rows, vocabulary, dtype))
    assert blocks(x) == size
    u = torch.rand(rows, generator=torch.Generator().manual_seed(9))
    check(x, u)
    check(x, u, top_k=in_turn([1, 2, 3, 40, 0, 5], rows), temperature=in_turn([0, 1, 2, 1, 1, 0.0], rows))


@pytest.mark.parametrize("vocabulary,size", [(2500, 1), (9999, 2), (20000, 4), (40000, 8)])
def test_extremes_of_the_types(vocabulary, size):
    for dtype, values in ((BF16, [[3.3895e38, -3.3895e38, 1e30, 0.0, 3.3895e38], [1e-40, -1e-40, 0.0, 2e-40, 1e-38]]),
                          (FP16, [[65504.0, -65504.0, 6e4, 0.0, 65504.0], [6e-8, -6e-8, 0.0, 1.2e-7, 6e-5]])):
        for fill in (-INF, torch.finfo(dtype).min, 0.0):
            x = torch.full((2, vocabulary), fill, dtype=dtype)
            x[:, ::vocabulary // 5][:, :5] = torch.tensor(values, dtype=dtype)
            for t in (1.0, 1e-30, 1e38):
                check(x, [0.7, 0.3], temperature=[t, t])
                check(x, [0.2, 0.9], temperature=[t, t], top_k=[3, 3])
                check(x, [0.99, 0.4], temperature=[t, t], top_k=[300, 2000], top_p=[0.9, 0.6])


@pytest.mark.parametrize("vocabulary,size", [(4097, 1), (9999, 2), (20000, 4), (151936, 8)])
@pytest.mark.parametrize("many", [1, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 512, 513, 1023, 1024, 1025])
def test_lists_of_every_size(vocabulary, size, many):
    """Exactly `many` tokens that are not masked, spread over all blocks' runs. Equal ones are all listed, whatever top-k is; up to
    1024 of them are put in order there, places being counted up to 256, and more go to the histogram. Different ones are all
    listed where top-k is as large as their number."""
    rows, g = 3, torch.Generator().manual_seed(many)
    equal = torch.full((rows, vocabulary), -INF, dtype=FP16)
    different = equal.clone()
    for i in range(rows):
        places = torch.cat([torch.tensor([0, vocabulary - 1]), 1 + torch.randperm(vocabulary - 2, generator=g)])[:many]
        equal[i, places] = 1.5
        different[i, places] = (torch.randn(many, generator=g) * 3).half()
    assert blocks(equal) == size
    u = [0.0, 1 - 2.0 ** -24, 0.61]
    for top_k in (256, min(256, many), max(1, min(255, many - 1)), max(1, min(256, many // 2))):
        check(equal, u, top_k=[top_k] * rows)
        check(different, u, top_k=[top_k] * rows)
    check(different, u, top_k=[256] * rows, top_p=[0.9, 0.5, 0.99], min_p=[0.0, 0.01, 0.001], temperature=[3.0, 1.0, 0.5])
    check(equal, u, top_k=[256] * rows, top_p=[0.9, 0.5, 0.99])
    check(equal, u, temperature=[0.0, 1.0, 0.0], top_k=[0, 1, 2])


@pytest.mark.parametrize("low", [-INF, None])
@pytest.mark.parametrize("many", [0, 65535, 65536, 70000])
def test_overflowing_counters_beside_many_groups(many, low):
    """Fp16, a block a row, hundreds of groups of 32 values, which a thread each sums up as a series: beside a value that more logits
    have than 16 bits count, and beside masks of either kind."""
    vocabulary, rows, g = 100_003, 76, torch.Generator().manual_seed(many)
    base = randn(many, 4, vocabulary, FP16, 3.0)
    for i in range(4):
        places = torch.randperm(vocabulary, generator=g)
        base[i, places[:many]] = [1.0, -0.0, 3.0, -2.0][i]
        base[i, places[many:many + 300]] = [1.0009765625, 0.0, 2.998046875, -2.001953125][i]  # its neighbour
        base[i, places[many + 1000:many + [0, 10000, 25000, 29000][i]]] = torch.finfo(FP16).min if low is None else low
    x = base.repeat(rows // 4, 1)
    assert blocks(x) == 1
    keys = x[0][x[0] > -60000].view(torch.int16).to(torch.int32) >> 5
    assert len(keys.unique()) > 192
    u = torch.rand(rows, generator=g)
    check(x, u)
    check(x, u, temperature=in_turn([0.5, 1.0, 4.0, 30.0, INF], rows), top_p=in_turn([0.9, 0.3, 0.999], rows),
          min_p=in_turn([0.0, 0.01], rows))
    check(x, u, top_k=in_turn([300, 5000, 70000, 99999], rows), temperature=in_turn([1.0, 50.0], rows))


@pytest.mark.parametrize("vocabulary,rows,size", [(9999, 12, 2), (20000, 12, 4), (151936, 12, 8), (9999, 160, 1)])
def test_captured_with_other_numbers(vocabulary, rows, size):
    """Replayed with rows that have an answer, none, a list too long and other settings."""
    x, u = randn(3, rows, vocabulary, BF16).cuda(), torch.rand(rows, device="cuda")
    given = dict(temperature=torch.ones(rows, device="cuda"), top_k=torch.zeros(rows, dtype=torch.int32, device="cuda"),
                 top_p=torch.ones(rows, device="cuda"), min_p=torch.zeros(rows, device="cuda"))
    K.sample(x, u, **given)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens, logprobs = K.sample(x, u, **given)
    for seed in range(4):
        now = settings(seed + rows, rows)
        new = randn(seed, rows, vocabulary, BF16)
        new[seed], new[seed + 4, vocabulary - 1 - seed], new[seed + 8] = 2.0, NAN, -INF
        x.copy_(new)
        u.copy_(torch.rand(rows, generator=torch.Generator().manual_seed(seed)))
        for name, t in given.items():
            t.copy_(torch.tensor(now[name]))
        graph.replay()
        want = check(new, u.cpu(), **now)
        assert torch.equal(tokens, want[0]) and torch.equal(logprobs, want[1])
