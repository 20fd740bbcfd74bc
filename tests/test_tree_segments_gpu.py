"""Trees over contexts with many more key tiles than thread blocks: long segments of either kind, parts that
begin and end inside a sequence, accumulators rescaled on the way."""

import math

import pytest
import torch

from tests._serving import attend, check
from tests.test_serving_attention_gpu import BF16, FP16, as_int64, chain_sets, make_cache, randn
from xpu_playground_b200 import kernels as K

pytestmark = pytest.mark.gpu
LENS = [1500 + 173 * i % 2500 for i in range(16)]


def run(counts, q_heads, kv_heads, d, dtype, seed, heads, rise=0.0, heat=1.0, spoil=None, size=64):
    """rise: how far scores rise over 4000 positions, on average."""
    cache, flat = make_cache(LENS, kv_heads, d, size, dtype, seed)
    nodes, group = sum(counts), q_heads // kv_heads
    q = randn(seed + 50, nodes, q_heads, d, dtype=dtype, scale=heat)
    k, v = randn(seed + 51, nodes, kv_heads, d, dtype=dtype), randn(seed + 52, nodes, kv_heads, d, dtype=dtype)
    if rise:
        q[:, :, 0] = math.sqrt(d) / 8
        for i, n in enumerate(LENS):
            slope = (torch.arange(n, device="cuda") * (8 * rise / 4000)).to(dtype)
            flat[i][0][:, :, 0] = slope[:, None]
            for p in range(-(-n // size)):
                m = min(size, n - p * size)
                cache.k[1, cache.tables[i, p].long(), :, :m, 0] = slope[p * size:p * size + m]
        k[:, :, 0] = 8 * rise * 0.6
    sets = chain_sets(counts, seed)
    if spoil is not None:
        v[spoil[0], :, 9] = spoil[1]
    starts = torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=torch.int32, device="cuda")
    ids = torch.arange(16, dtype=torch.int32, device="cuda")
    ws = K.tree_attention_workspace(16, nodes, q_heads, kv_heads, d)
    args = (cache, 1, ids, starts, as_int64(sets), q, k, v, ws)
    out, lse = K.tree_attention(*args)
    for _ in range(3):
        again = K.tree_attention(*args)
        assert torch.equal(out.view(torch.int16), again[0].view(torch.int16)) and torch.equal(lse, again[1])
    some = [i for i in range(16) if i % 5 == 0 or spoil is not None and int(starts[i]) <= spoil[0] < int(starts[i + 1])]
    for i in some:
        at = slice(int(starts[i]), int(starts[i + 1]))
        n = counts[i]
        allowed = torch.cat([torch.ones(n, LENS[i], dtype=torch.bool),
                             torch.tensor([[b >> j & 1 for j in range(n)] for b in sets[at]], dtype=torch.bool).view(n, n)], 1)
        keys, values = (torch.cat([a.cpu(), b[at].cpu()]) for a, b in ((flat[i][0], k), (flat[i][1], v)))
        for h in heads:
            want = attend(q[at, h].cpu(), keys[:, h // group], values[:, h // group], allowed, 1 / math.sqrt(d))
            check(out[at, h], lse[at, h], *want, dtype)
    assert cache.status() == 0 and K.device_status() == 0


MANY, FEW = [64] * 16, [1 + 5 * i % 20 for i in range(16)]
MIXED = [[64, 33, 1, 20][i % 4] for i in range(16)]


@pytest.mark.parametrize("d,dtype", [(128, BF16), (64, FP16), (128, FP16), (64, BF16)])
@pytest.mark.parametrize("counts", [MANY, FEW, MIXED])
def test_long_segments(counts, d, dtype):
    run(counts, 32, 8, d, dtype, 200, [0, 13, 31])


@pytest.mark.parametrize("d,dtype", [(128, FP16), (64, BF16)])
@pytest.mark.parametrize("counts", [MANY, FEW])
@pytest.mark.parametrize("rise", [60.0, -60.0])
def test_long_segments_with_rising_and_falling_scores(counts, d, dtype, rise):
    run(counts, 32, 8, d, dtype, 210, [2, 30], rise=rise)


@pytest.mark.parametrize("counts", [MANY, FEW])
def test_long_segments_with_peaked_scores(counts):
    run(counts, 32, 8, 64, BF16, 220, [1, 17], heat=20.0)


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("counts,node", [(MANY, 64 * 5 + 3), (FEW, 60), (MIXED, 70)])
def test_long_segments_with_a_non_finite_draft(counts, node, value):
    """Beside rows that do not attend it, in the same tile: those come out as if it were not there."""
    run(counts, 32, 8, 128, BF16, 230, [4, 29], spoil=(node, value))


@pytest.mark.parametrize("q_heads,kv_heads", [(28, 4), (14, 2), (8, 8), (16, 1)])
def test_long_segments_of_other_groupings(q_heads, kv_heads):
    run(MIXED, q_heads, kv_heads, 64, FP16, 240, [0, q_heads - 1], size=16)
