"""Attention over packed prompts and of drafted trees over the paged cache,
against a plain implementation in 64 bits at the sizes and masks where such
kernels go wrong."""

import math

import pytest
import torch

from tests._serving import attend, check
from xpu_playground_b200 import kernels as K
from xpu_playground_b200.kv_cache import BAD_INDEX, KvCache

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def randn(seed, *shape, dtype=BF16, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


# ---------------------------------------------------------------- prompts ----

def prompt_reference(lens, q, k, v, scale, heads=None):
    group = q.shape[1] // k.shape[1]
    q, k, v = q.cpu(), k.cpu(), v.cpu()
    out = torch.zeros(q.shape, dtype=torch.float64)
    lse, size = torch.zeros(q.shape[:2], dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    at = 0
    for n in lens:
        mask = torch.ones(n, n, dtype=torch.bool).tril()
        for h in range(q.shape[1]) if heads is None else heads:
            s = slice(at, at + n)
            out[s, h], lse[s, h], size[s, h] = attend(q[s, h], k[s, h // group], v[s, h // group], mask, scale)
        at += n
    return out, lse, size


def run_prompt(lens, q_heads, kv_heads, d, dtype, seed=0, heat=1.0, scale=None):
    tokens = sum(lens)
    q, k, v = (randn(seed + i, tokens, h, d, dtype=dtype, scale=heat if i == 0 else 1.0)
               for i, h in enumerate((q_heads, kv_heads, kv_heads)))
    plan = K.PromptPlan(lens, q_heads, kv_heads, d)
    out, lse = K.prompt_attention(plan, q, k, v, scale=scale)
    want = prompt_reference(lens, q, k, v, 1 / math.sqrt(d) if scale is None else scale)
    check(out, lse, want[0], want[1], want[2], dtype)
    assert K.device_status() == 0


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("q_heads,kv_heads,d", [(4, 1, 128), (2, 2, 64), (7, 1, 128), (6, 2, 64), (16, 1, 64), (3, 3, 128)])
def test_prompt_heads_and_types(q_heads, kv_heads, d, dtype):
    run_prompt([1, 130, 0, 33, 257], q_heads, kv_heads, d, dtype)


@pytest.mark.parametrize("lens", [[1], [2], [31], [32], [63], [64], [65], [127], [128], [129], [255], [256], [300], [513],
                                  [0, 1], [1] * 40, [0, 0, 5, 0], [1, 64, 1, 128, 1]])
def test_prompt_lengths(lens):
    run_prompt(lens, 4, 1, 128, BF16, seed=len(lens))


@pytest.mark.parametrize("q_heads,kv_heads", [(64, 1), (40, 1), (12, 4)])
def test_prompt_wide_groups(q_heads, kv_heads):
    run_prompt([70, 3], q_heads, kv_heads, 64, BF16, seed=3)


def test_prompt_peaked_scores_and_scale():
    """Rows whose maximum jumps late and far: every rescale of the running softmax."""
    run_prompt([700], 2, 1, 128, BF16, seed=5, heat=20.0)
    run_prompt([200], 2, 1, 64, FP16, seed=6, scale=0.5)


def test_prompt_rising_maximum():
    n, d = 640, 64
    q = torch.ones(n, 1, d, dtype=BF16, device="cuda")
    k = (torch.arange(n, device="cuda")[:, None, None] / 16.0).expand(n, 1, d).to(BF16).contiguous()
    v = randn(1, n, 1, d)
    out, lse = K.prompt_attention(K.PromptPlan([n], 1, 1, d), q, k, v)
    want = prompt_reference([n], q, k, v, 1 / 8.0)
    check(out, lse, *want, BF16)


def test_prompt_many_blocks_many_items():
    """More tiles than thread blocks: every block runs several."""
    lens = [100, 900, 333, 1, 512] * 2
    q, k, v = (randn(20 + i, sum(lens), h, 64, dtype=FP16) for i, h in enumerate((16, 8, 8)))
    out, lse = K.prompt_attention(K.PromptPlan(lens, 16, 8, 64), q, k, v)
    heads = [0, 3, 15]
    want = prompt_reference(lens, q, k, v, 1 / 8.0, heads)
    check(out[:, heads], lse[:, heads], *(w[:, heads] for w in want), FP16)


def test_prompt_strided_rows_and_given_outputs():
    """q, k and v as slices of one fused projection, outputs inside a wider buffer, on a stream of its own."""
    lens, qh, kvh, d = [90, 41], 4, 2, 128
    n = sum(lens)
    fused = randn(9, n, qh + 2 * kvh, d)
    q, k, v = fused[:, :qh], fused[:, qh:qh + kvh], fused[:, qh + kvh:]
    wide = torch.full((n, qh + 1, d), 7.0, dtype=BF16, device="cuda")
    lse = torch.empty(n, qh, device="cuda")
    plan = K.PromptPlan(lens, qh, kvh, d)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        K.prompt_attention(plan, q, k, v, out=wide[:, :qh], lse=lse)
    s.synchronize()
    want = prompt_reference(lens, q, k, v, 1 / math.sqrt(d))
    check(wide[:, :qh], lse, *want, BF16)
    assert bool((wide[:, qh] == 7.0).all())


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("where", [(0, 3), (63, 64), (199, 5), (300, 310)])
def test_prompt_non_finite_values_reach_only_rows_that_attend_them(value, where):
    """A non-finite key or value of position j leaves rows before j, and the
    other prompts of the batch, as they are."""
    lens, d = [200, 130], 64
    q, k, v = (randn(30 + i, sum(lens), h, d) for i, h in enumerate((2, 1, 1)))
    a, b = where
    v[a, 0, 7] = value
    k[b, 0] = value
    out, lse = K.prompt_attention(K.PromptPlan(lens, 2, 1, d), q, k, v)
    clean_k, clean_v = k.clone(), v.clone()
    clean_k[b], clean_v[a, 0, 7] = 0, 0
    want = prompt_reference(lens, q, clean_k, clean_v, 1 / 8.0)
    spoilt = torch.zeros(sum(lens), d, dtype=torch.bool)
    owner = lambda t: (0, 200) if t < 200 else (200, 330)  # noqa: E731
    spoilt[a:owner(a)[1], 7] = True
    spoilt[b:owner(b)[1]] = True
    good = ~spoilt[:, None, :].expand(-1, 2, -1)
    assert torch.isfinite(out.float()).cpu()[good].all()
    err = (out.double().cpu() - want[0]).abs()
    tol = 2.0 ** -8 * (want[0].abs() + 1.1 * want[2]) + 1e-5
    assert (err <= tol)[good].all()
    # the rows that attend a non-finite value show it (a value of weight zero gives 0 x inf = NaN as well)
    assert not torch.isfinite(out[a:owner(a)[1], :, 7].float()).any()


def test_prompt_repeats_bit_for_bit():
    lens = [500, 77]
    q, k, v = (randn(40 + i, sum(lens), h, 128) for i, h in enumerate((8, 2, 2)))
    plan = K.PromptPlan(lens, 8, 2, 128)
    first = K.prompt_attention(plan, q, k, v)
    for _ in range(5):
        again = K.prompt_attention(plan, q, k, v)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


# ------------------------------------------------------------------ trees ----

def make_cache(lens, kv_heads, d, size, dtype, seed, layers=2, fill=math.nan):
    """A cache whose pages lie in random order; everything not in use holds `fill`."""
    g = torch.Generator().manual_seed(seed)
    used = [-(-n // size) for n in lens]
    pages = sum(used) + 3
    order = torch.randperm(pages, generator=g)
    cache = KvCache(layers, pages, size, kv_heads, d, len(lens), max(max(lens), 1) + size, dtype=dtype)
    cache.k.fill_(fill)
    cache.v.fill_(fill)
    flat = []
    at = 0
    for i, n in enumerate(lens):
        k, v = randn(seed + 2 * i + 1, n, kv_heads, d, dtype=dtype), randn(seed + 2 * i + 2, n, kv_heads, d, dtype=dtype)
        for p in range(used[i]):
            page, m = int(order[at]), min(size, n - p * size)
            at += 1
            cache.tables[i, p] = page
            cache.refs[page] = 1
            cache.k[1, page, :, :m] = k[p * size:p * size + m].transpose(0, 1)
            cache.v[1, page, :, :m] = v[p * size:p * size + m].transpose(0, 1)
        flat.append((k, v))
    cache.lens.copy_(torch.tensor(lens, dtype=torch.int32))
    return cache, flat


def chain_sets(counts, seed):
    g = torch.Generator().manual_seed(seed)
    sets = []
    for n in counts:
        tree = []
        for i in range(n):
            parent = int(torch.randint(-1, i, (1,), generator=g)) if i else -1
            tree.append((tree[parent] if parent >= 0 else 0) | 1 << i)
        sets += tree
    return sets


def as_int64(sets):
    return torch.tensor([s - (1 << 64) if s >> 63 else s for s in sets], dtype=torch.int64, device="cuda")


def run_tree(lens, counts, q_heads, kv_heads, d, size, dtype=BF16, seed=100, sets=None, order=None, fill=math.nan, heat=1.0,
             repeat=1):
    cache, flat = make_cache(lens, kv_heads, d, size, dtype, seed, fill=fill)
    order = list(range(len(lens))) if order is None else order
    nodes = sum(counts)
    q = randn(seed + 50, nodes, q_heads, d, dtype=dtype, scale=heat)
    k, v = randn(seed + 51, nodes, kv_heads, d, dtype=dtype), randn(seed + 52, nodes, kv_heads, d, dtype=dtype)
    sets = chain_sets(counts, seed) if sets is None else sets
    starts = torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=torch.int32, device="cuda")
    ids = torch.tensor(order, dtype=torch.int32, device="cuda")
    ws = K.tree_attention_workspace(len(order), nodes, q_heads, kv_heads, d)
    out, lse = K.tree_attention(cache, 1, ids, starts, as_int64(sets), q, k, v, ws)
    for _ in range(repeat):
        again = K.tree_attention(cache, 1, ids, starts, as_int64(sets), q, k, v, ws)
        assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
    want, want_lse = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape[:2], dtype=torch.float64)
    sizes, group, at = torch.zeros(q.shape, dtype=torch.float64), q_heads // kv_heads, 0
    for i, n in zip(order, counts):
        s = slice(at, at + n)
        mask = torch.cat([torch.ones(n, lens[i], dtype=torch.bool),
                          torch.tensor([[b >> j & 1 for j in range(n)] for b in sets[s]], dtype=torch.bool).view(n, n)], 1)
        keys, values = (torch.cat([a.cpu(), b[s].cpu()]) for a, b in ((flat[i][0], k), (flat[i][1], v)))
        for h in range(q_heads):
            want[s, h], want_lse[s, h], sizes[s, h] = attend(q[s, h].cpu(), keys[:, h // group], values[:, h // group], mask,
                                                             1 / math.sqrt(d))
        at += n
    check(out, lse, want, want_lse, sizes, dtype)
    assert cache.status() == 0 and K.device_status() == 0
    return out


@pytest.mark.parametrize("size", [16, 32, 64, 128])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_tree_pages_and_types(size, dtype):
    run_tree([0, 1, size - 1, size, size + 1, 130, 300], [3, 1, 5, 2, 9, 1, 4], 4, 2, 128, size, dtype)


@pytest.mark.parametrize("q_heads,kv_heads,d", [(1, 1, 64), (7, 1, 128), (6, 2, 64), (16, 1, 64), (3, 3, 128), (64, 1, 64)])
def test_tree_heads(q_heads, kv_heads, d):
    run_tree([77, 140], [11, 2], q_heads, kv_heads, d, 16, seed=7)


@pytest.mark.parametrize("nodes", [1, 2, 31, 32, 33, 63, 64])
def test_tree_node_counts(nodes):
    run_tree([200, 15], [nodes, 64], 4, 1, 64, 32, seed=nodes)


@pytest.mark.parametrize("length", [1, 2, 127, 128, 129, 255, 256, 257, 1000, 2500])
def test_tree_single_token_lengths(length):
    run_tree([length], [1], 8, 2, 128, 16, seed=length)


def test_tree_many_sequences_and_order():
    lens = [i * 37 % 400 for i in range(40)]
    run_tree(lens, [i % 5 for i in range(40)], 4, 2, 64, 16, seed=11, order=[(i * 7) % 40 for i in range(40)])


def test_tree_long_context_is_split():
    run_tree([9000, 3], [20, 3], 4, 1, 128, 64, seed=13)


def test_tree_rows_that_attend_nothing():
    """No context and an empty set: zeros and -inf, beside rows that see one node."""
    out = run_tree([0, 0, 20], [4, 1, 3], 4, 2, 64, 16, sets=[0, 2, 0, 9, 0, 0, 3, 4], seed=17)
    assert not out[0].any() and not out[2].any() and not out[4].any()


def test_tree_peaked_scores():
    run_tree([600], [30], 4, 1, 64, 16, seed=19, heat=20.0)


@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_tree_non_finite_drafts_reach_only_nodes_that_attend_them(value):
    """Node 2's key and value are not finite; only nodes whose set names it see them."""
    cache, flat = make_cache([40], 1, 64, 16, BF16, 23)
    sets = [1, 3, 5, 9, 13, 17]  # node 4 attends 0, 2, 3; node 2 itself; no other attends 2
    q, k, v = randn(1, 6, 2, 64), randn(2, 6, 1, 64), randn(3, 6, 1, 64)
    starts, ids = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 6], [0]))
    ws = K.tree_attention_workspace(1, 6, 2, 1, 64)
    clean = K.tree_attention(cache, 1, ids, starts, as_int64(sets), q, k, v, ws)
    k[2, 0], v[2, 0] = value, value
    out, lse = K.tree_attention(cache, 1, ids, starts, as_int64(sets), q, k, v, ws)
    for r in (0, 1, 3, 5):
        assert torch.equal(out[r], clean[0][r]) and torch.equal(lse[r], clean[1][r])
    for r in (2, 4):
        assert not torch.isfinite(out[r].float()).any()


def test_tree_bad_indices_are_reported_and_read_as_nothing():
    cache, flat = make_cache([40, 40], 1, 64, 16, BF16, 29)
    cache.tables[0, 1] = 10 ** 6  # the pool has fewer pages
    q, k, v = randn(1, 2, 2, 64), randn(2, 2, 1, 64), randn(3, 2, 1, 64)
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    ws = K.tree_attention_workspace(2, 2, 2, 1, 64)
    ids = torch.tensor([0, 77], dtype=torch.int32, device="cuda")  # and sequence 77 does not exist
    out, lse = K.tree_attention(cache, 1, ids, starts, as_int64([1, 1]), q, k, v, ws)
    assert cache.status() == BAD_INDEX and cache.status() == 0
    assert torch.equal(out[1], v[1].expand(2, 64))  # no context: the node itself


def test_tree_matches_prompt_attention():
    """A chain of drafts over a cached prefix gives what one prompt gives at those positions."""
    n, extra, d = 150, 40, 128
    q, k, v = (randn(60 + i, n + extra, h, d) for i, h in enumerate((4, 2, 2)))
    whole, whole_lse = K.prompt_attention(K.PromptPlan([n + extra], 4, 2, d), q, k, v)
    cache = KvCache(1, 20, 16, 2, d, 1, 200)
    ids, starts = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0], [0, n]))
    cache.append(ids, starts, k[None, :n], v[None, :n])
    sets = as_int64([(1 << (i + 1)) - 1 for i in range(extra)])
    ws = K.tree_attention_workspace(1, extra, 4, 2, d)
    starts = torch.tensor([0, extra], dtype=torch.int32, device="cuda")
    out, lse = K.tree_attention(cache, 0, ids, starts, sets, q[n:].contiguous(), k[n:], v[n:], ws)
    assert (lse - whole_lse[n:]).abs().max() < 2e-4
    assert (out.float() - whole[n:].float()).abs().max() < 4 * 2.0 ** -8


def test_python_argument_checks():
    plan = K.PromptPlan([8], 2, 1, 64)
    q, k = randn(1, 8, 2, 64), randn(2, 8, 1, 64)
    with pytest.raises(ValueError):
        K.prompt_attention(plan, q[:4], k, k)
    with pytest.raises(ValueError):
        K.prompt_attention(plan, q, k.half(), k)
    with pytest.raises(ValueError):
        K.prompt_attention(plan, q.transpose(0, 1).contiguous().transpose(0, 1), k, k)
    with pytest.raises(ValueError):
        K.prompt_attention(plan, q.cpu(), k, k)
    cache, _ = make_cache([4], 1, 64, 16, BF16, 1)
    ws = K.tree_attention_workspace(1, 8, 2, 1, 64)
    ids, starts = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0], [0, 8]))
    with pytest.raises(ValueError):
        K.tree_attention(cache, 0, ids.long(), starts, as_int64([1] * 8), q, k, k, ws)
    with pytest.raises(ValueError):
        K.tree_attention(cache, 0, ids, starts, as_int64([1] * 7), q, k, k, ws)
    with pytest.raises(K._lib.XpuError, match="layer"):
        K.tree_attention(cache, 5, ids, starts, as_int64([1] * 8), q, k, k, ws)
    with pytest.raises(K._lib.XpuError, match="null pointer"):
        K.tree_attention(cache, 0, ids, starts, as_int64([1] * 8), q, k, k, ws[:0])
