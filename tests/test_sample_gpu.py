"""Sampling against a sort in 64 bits: the same tokens, whatever the settings."""

import numpy as np
import pytest
import torch

from tests._fp8 import choose
from xpu_playground_b200 import kernels as K

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16
INF, NAN = float("inf"), float("nan")


def check(logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    rows = len(logits)
    lists = dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    given = {n: torch.tensor(v, dtype=torch.int32 if n == "top_k" else torch.float32) for n, v in lists.items() if v is not None}
    u = torch.as_tensor(u, dtype=torch.float32)
    tokens, logprobs = K.sample(logits.cuda(), u.cuda(), **{n: t.cuda() for n, t in given.items()})
    host = logits.cpu().double().numpy()
    want = [choose(host[i], float(u[i]), **{n: t[i].item() for n, t in given.items()}) for i in range(rows)]
    assert tokens.tolist() == [t for t, _ in want]
    p = np.array([x for _, x in want])
    got, fine = logprobs.double().cpu().numpy(), np.isfinite(p)
    assert np.array_equal(got[~fine], p[~fine])
    # one rounding to FP32; the sums are FP64
    assert (np.abs(got[fine] - p[fine]) <= 2.0 ** -24 * np.abs(p[fine]) + 1e-10).all()
    return tokens, logprobs


def randn(seed, rows, vocabulary, dtype, size=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocabulary, generator=g) * size
    x += 10 * torch.rand(rows, vocabulary, generator=g) * (torch.rand(rows, vocabulary, generator=g) < 20 / vocabulary)
    return x.to(dtype)


def settings(seed, rows):
    r = np.random.RandomState(seed)
    return dict(temperature=r.choice([0.0, 0.01, 0.5, 0.7, 1.0, 1.0, 1.7, 30.0], rows).tolist(),
                top_k=r.choice([0, 0, 1, 2, 20, 50, 255, 256, 257, 1000, 1 << 30], rows).tolist(),
                top_p=r.choice([1.0, 1.0, 0.999, 0.95, 0.8, 0.5, 0.01, 0.0], rows).tolist(),
                min_p=r.choice([0.0, 0.0, 1e-4, 0.05, 0.3, 1.0], rows).tolist())


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("rows,vocabulary", [(5, 1), (40, 2), (60, 7), (60, 31), (60, 33), (100, 1000), (100, 4097), (30, 65536),
                                             (1, 151936), (3, 151936), (16, 151936), (20, 151936), (40, 100003), (80, 151936), (200, 9999),
                                             (2, 300000), (20, 1 << 20)])
def test_tokens(rows, vocabulary, dtype):
    u = torch.rand(rows, generator=torch.Generator().manual_seed(rows))
    check(randn(vocabulary, rows, vocabulary, dtype), u, **settings(rows + vocabulary, rows))


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_defaults(dtype):
    check(randn(1, 50, 3000, dtype), torch.rand(50, generator=torch.Generator().manual_seed(1)))


@pytest.mark.parametrize("vocabulary", [64, 5000, 151936])
def test_equal_logits_go_by_their_ids(vocabulary):
    """All weights 1: the sums are whole numbers, and token i is chosen from u = i / n on."""
    n = 64
    u = (torch.arange(n) / n).float()
    tokens, _ = check(torch.full((n, vocabulary), -3.0, dtype=BF16), u)
    assert tokens.tolist() == [i * vocabulary // n for i in range(n)]
    check(torch.full((n, vocabulary), 0.5, dtype=BF16), u, top_p=[0.5] * n)
    check(torch.full((n, vocabulary), 0.5, dtype=FP16), u, top_k=[max(1, i * 37 % vocabulary) for i in range(n)])
    check(torch.full((n, vocabulary), 0.5, dtype=FP16), u, top_p=[0.25] * n, min_p=[1.0] * n, temperature=[0.3] * n)


def test_zeros_of_both_signs_are_equal():
    x = torch.zeros(32, 1001, dtype=BF16)
    x[:, ::3] = -0.0
    u = (torch.arange(32) / 32).float()
    check(x, u, top_k=[0, 1, 2, 500] * 8)
    check(x.half(), u, temperature=[0.0, 1.0] * 16)


@pytest.mark.parametrize("many", [65535, 65536, 65537, 70000, 131072, 151900])
@pytest.mark.parametrize("values", [(1.0, 1.0078125), (1.0078125, 1.015625), (-2.0, 4.0), (0.0, -5.0)])
def test_more_equal_logits_than_16_bits_count(many, values):
    """Neighbouring values share a counter's word."""
    rows, g = 200, torch.Generator().manual_seed(many)
    x = randn(3, 1, 151936, BF16).repeat(rows, 1)
    x[:, torch.randperm(151936, generator=g)[:many]] = values[0]
    x[:, torch.randperm(151936, generator=g)[:66000]] = values[1]
    check(x, torch.rand(rows, generator=g), **settings(many, rows))
    check(x[:3], torch.rand(3, generator=g), **settings(many, 3))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("low", [-INF, None])
@pytest.mark.parametrize("vocabulary", [50, 151936])
def test_masks(dtype, low, vocabulary):
    rows, g = 24, torch.Generator().manual_seed(2)
    x = randn(4, rows, vocabulary, dtype)
    low = torch.finfo(dtype).min if low is None else low
    for i in range(rows):
        x[i, torch.rand(vocabulary, generator=g) < [0.1, 0.9, 0.999, 1.0][i % 4]] = low
    x[3::8, vocabulary // 3] = -1.0  # one token left; the other rows of this kind have none
    u = torch.rand(rows, generator=g)
    tokens, logprobs = check(x, u, **settings(5, rows))
    check(x, u)
    if low == -INF:
        chosen = tokens.cpu().long()
        assert all(t == -1 or x[i, t] > -INF for i, t in enumerate(chosen)) and (chosen[7::8] == -1).all()


def test_rows_that_are_not_numbers():
    x = randn(5, 10, 2000, BF16)
    x[1, 7], x[2, 1999], x[3, 0], x[4, :] = NAN, INF, -NAN, -INF
    x[5, 3:] = -INF
    x.view(torch.int16)[6, 9] = -1  # a negative NaN
    check(x, [0.5] * 10)
    check(x, [0.5] * 10, temperature=[0.0] * 10)
    check(x, [0.5] * 10, top_k=[3] * 10)


def test_settings_that_are_not_numbers():
    x = randn(6, 12, 500, BF16)
    check(x, [0.1, -0.1, 1.0, NAN, INF, 0.5, 0.5, 0.5, 0.5, 0.5, 0.5, 0.5],
          temperature=[1, 1, 1, 1, 1, NAN, -1.0, 1, 1, 1, INF, 1e-40], top_k=[0, 0, 0, 0, 0, 0, 0, -1, 0, 0, 0, 0],
          top_p=[1, 1, 1, 1, 1, 1, 1, 1, NAN, 1, 1, 1], min_p=[0, 0, 0, 0, 0, 0, 0, 0, 0, NAN, 0, 0])
    # beyond their range: as if at its end
    check(x, [0.3] * 12, top_p=[-1.0, 0.0, 2.0] * 4, min_p=[-1.0, 5.0, 1.0, 0.0] * 3)


@pytest.mark.parametrize("u", [0.0, 2.0 ** -24, 0.5, 1.0 - 2.0 ** -24])
def test_ends_of_u(u):
    for vocabulary in (1, 100, 151936):
        check(randn(7, 8, vocabulary, BF16), [u] * 8, **settings(8, 8))
        check(randn(7, 8, vocabulary, BF16), [u] * 8)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("shift", range(8))
def test_rows_at_any_address(dtype, shift):
    held = randn(9, 6, 1013, dtype).cuda()
    x = held[:, shift:shift + 1000]
    u = torch.rand(6, generator=torch.Generator().manual_seed(9))
    check(x, u)
    check(x, u, top_k=[1, 2, 3, 40, 0, 5], temperature=[0, 1, 2, 1, 1, 0.0])


def test_extremes_of_the_types():
    x = torch.tensor([[3.3895e38, -3.3895e38, 1e30, 0.0, 3.3895e38], [1e-40, -1e-40, 0.0, 2e-40, 1e-38]], dtype=BF16)
    for t in (1.0, 1e-30, 1e38):
        check(x, [0.7, 0.3], temperature=[t, t])
        check(x, [0.2, 0.9], temperature=[t, t], top_k=[3, 3])


def test_frequencies_are_the_probabilities():
    """Tokens of a fine grid of u: each as often as its probability says, to one step of the grid."""
    n, x = 4096, torch.tensor([0.5, 2.0, -1.0, 1.0], dtype=BF16)
    tokens, _ = K.sample(x.repeat(n, 1).cuda(), ((torch.arange(n) + 0.5) / n).cuda())
    p = torch.softmax(x.double(), 0)
    assert (torch.bincount(tokens.long().cpu(), minlength=4).double() / n - p).abs().max() <= 1 / n


def test_given_outputs_no_rows_and_repeats():
    x, u = randn(10, 300, 151936, BF16).cuda(), torch.rand(300, generator=torch.Generator().manual_seed(4)).cuda()
    tokens, logprobs = torch.full((301,), 7, dtype=torch.int32, device="cuda"), torch.full((301,), 7.0, device="cuda")
    got = K.sample(x, u, tokens=tokens[:300], logprobs=logprobs[:300])
    assert int(tokens[300]) == 7 and float(logprobs[300]) == 7
    for _ in range(3):
        again = K.sample(x, u)
        assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])
    few = K.sample(x[:5], u[:5])  # another number of blocks a row: the same tokens
    assert torch.equal(few[0], got[0][:5]) and (few[1] - got[1][:5]).abs().max() <= 2.0 ** -20
    assert K.sample(x[:0], u[:0])[0].shape == (0,)
