"""What single values do in the serving attention: infinities and NaN that a row attends,
finite columns beside them, and weights far below the largest."""

import math

import pytest
import torch

from tests._serving import UNIT, attend, check
from tests.test_serving_attention_gpu import BF16, FP16, as_int64, make_cache, prompt_reference, randn
from xpu_playground_b200 import kernels as K
from xpu_playground_b200.kv_cache import KvCache

pytestmark = pytest.mark.gpu


def starts_of(counts):
    return torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("heads", [(1, 1), (4, 2)])
def test_prompt_columns_beside_non_finite_ones_are_rounded_once(heads):
    """Column 0 of every value is NaN, the others are near 0.3: each weight is far below half a
    step of the sum in 16 bits."""
    n, d = 1000, 64
    q, k = (randn(70 + i, n, h, d, scale=0.1) for i, h in enumerate(heads))
    v = (randn(72, n, heads[1], d).float() * 0.05 + 0.3).bfloat16()
    v[:, :, 0] = math.nan
    out, lse = K.prompt_attention(K.PromptPlan([n], *heads, d), q, k, v)
    want = prompt_reference([n], q, k, v, 1 / 8.0)
    check(out, lse, *want, BF16)


@pytest.mark.parametrize("length,nodes", [(0, 40), (90, 64), (700, 9)])
def test_tree_columns_beside_non_finite_ones_are_rounded_once(length, nodes):
    d = 128
    cache, flat = make_cache([length], 1, d, 16, BF16, 74)
    q, k = randn(75, nodes, 4, d, scale=0.1), randn(76, nodes, 1, d, scale=0.1)
    v = (randn(77, nodes, 1, d).float() * 0.05 + 0.3).bfloat16()
    v[:, 0, 3] = math.nan
    sets = [(1 << (i + 1)) - 1 for i in range(nodes)]
    ws = K.tree_attention_workspace(1, nodes, 4, 1, d)
    ids = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, lse = K.tree_attention(cache, 0 + 1, ids, starts_of([nodes]), as_int64(sets), q, k, v, ws)
    keys, values = (torch.cat([a.cpu(), b.cpu()])[:, 0] for a, b in ((flat[0][0], k), (flat[0][1], v)))
    allowed = torch.cat([torch.ones(nodes, length, dtype=torch.bool), torch.ones(nodes, nodes, dtype=torch.bool).tril()], 1)
    parts = [attend(q[:, h].cpu(), keys, values, allowed, 1 / math.sqrt(d)) for h in range(4)]
    check(out, lse, *(torch.stack(p, 1) for p in zip(*parts)), BF16)


@pytest.mark.parametrize("length", [200, 1000, 2040, 5000])
@pytest.mark.parametrize("value", [math.inf, -math.inf])
def test_attended_infinity_of_a_single_token_stays_one(length, value):
    """A draft's infinite value comes out in its column, whatever number of parts the sequence was cut into."""
    d = 128
    cache, flat = make_cache([length], 1, d, 16, BF16, 80)
    q, k, v = randn(81, 1, 4, d), randn(82, 1, 1, d), randn(83, 1, 1, d)
    v[0, 0, 5] = value
    ws = K.tree_attention_workspace(1, 1, 4, 1, d)
    ids = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, lse = K.tree_attention(cache, 1, ids, starts_of([1]), as_int64([1]), q, k, v, ws)
    keys, values = (torch.cat([a.cpu(), b.cpu()])[:, 0] for a, b in ((flat[0][0], k), (flat[0][1], v)))
    parts = [attend(q[:, h].cpu(), keys, values, torch.ones(1, length + 1, dtype=torch.bool), 1 / math.sqrt(d)) for h in range(4)]
    want, want_lse, size = (torch.stack(p, 1) for p in zip(*parts))
    assert bool((out[0, :, 5] == value).all())
    check(out, lse, want, want_lse, size, BF16)


def sink(keys, gap, at):
    """Keys and values of which number `at` is `gap` nats above the others and has value 0, the others 1:
    q = 8 e0, scale 1/8. The exact result is n w / (1 + n w) with w = exp(-gap)."""
    k, v = torch.zeros(keys, 1, 64, dtype=FP16, device="cuda"), torch.ones(keys, 1, 64, dtype=FP16, device="cuda")
    k[at, 0, 0], v[at] = gap, 0
    return k, v


def check_sink(out, lse, keys, gap):
    """Each weight is rounded to 2^-11 of itself or 2^-36 of the largest (fp16's smallest step is 2^-24, half of it
    2^-25, and the largest weight is held as 2^11 or more); 1e-4 for the FP32 arithmetic; then the output's own rounding."""
    others = (keys - 1) * math.exp(-gap)
    want = others / (1 + others)
    tol = (2 * UNIT[FP16] + 1e-4) * want + keys * 2.0 ** -36 + 2.0 ** -25
    assert float((out.double() - want).abs().max()) <= tol
    assert float((lse.double() - gap - math.log1p(others)).abs().max()) <= 1e-4


@pytest.mark.parametrize("gap", [8.0, 14.0, 17.5, 20.0])
@pytest.mark.parametrize("length,at", [(4095, 0), (4095, 4000), (16383, 7000), (65535, 0)])
def test_many_small_weights_beside_a_large_one_tree(gap, length, at):
    k, v = sink(length + 1, gap, at)
    cache = KvCache(1, 512, 128, 1, 64, 1, 65536, dtype=FP16)
    ids = torch.zeros(1, dtype=torch.int32, device="cuda")
    cache.append(ids, starts_of([length]), k[None, :length], v[None, :length])
    q = torch.zeros(1, 2, 64, dtype=FP16, device="cuda")
    q[:, :, 0] = 8
    ws = K.tree_attention_workspace(1, 1, 2, 1, 64)
    out, lse = K.tree_attention(cache, 0, ids, starts_of([1]), as_int64([1]), q, k[length:], v[length:], ws)
    check_sink(out, lse, length + 1, gap)
    assert cache.status() == 0


@pytest.mark.parametrize("gap", [8.0, 17.5])
@pytest.mark.parametrize("at", [0, 4000])
def test_many_small_weights_beside_a_large_one_prompt(gap, at):
    n = 8200
    k, v = sink(n, gap, at)
    q = torch.zeros(n, 2, 64, dtype=FP16, device="cuda")
    q[:, :, 0] = 8
    out, lse = K.prompt_attention(K.PromptPlan([n], 2, 1, 64), q, k, v)
    for row in (at, at + 1, at + 100, 6000, n - 1):
        check_sink(out[row], lse[row], row + 1, gap)
