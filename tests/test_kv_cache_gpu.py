"""The paged cache's operators against their definitions on the host: every
table, length, reference count and stored bit."""

import random

import numpy as np
import pytest
import torch

from tests._serving import HostCache
from xpu_playground_b200.kv_cache import BAD_INDEX, BAD_SEQUENCE, EXHAUSTED, SHARED_CUT, KvCache

pytestmark = pytest.mark.gpu


def ints(values):
    return torch.tensor(list(values), dtype=torch.int32, device="cuda")


def starts_of(counts):
    return ints([0] + list(np.cumsum(counts)))


def new_cache(layers=2, pages=40, size=16, kv_heads=2, d=64, sequences=8, positions=200, dtype=torch.bfloat16):
    cache = KvCache(layers, pages, size, kv_heads, d, sequences, positions, dtype=dtype)
    g = torch.Generator().manual_seed(pages)
    for pool in (cache.k, cache.v):
        pool.copy_(torch.randn(pool.shape, generator=g).to(dtype))
    return cache


def new_rows(cache, held, seed):
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn(cache.layers, held, cache.kv_heads, cache.head_dim, generator=g).to(cache.dtype) for _ in range(2))
    return k.cuda(), v.cuda(), *(t.view(torch.int16).numpy() for t in (k, v))


@pytest.mark.parametrize("size,kv_heads,d,dtype", [(16, 2, 64, torch.bfloat16), (32, 3, 128, torch.float16),
                                                   (64, 1, 64, torch.float16), (128, 2, 128, torch.bfloat16)])
def test_random_use(size, kv_heads, d, dtype):
    """A few hundred random requests, refused ones among them."""
    r = random.Random(size)
    cache = new_cache(layers=2, pages=24, size=size, kv_heads=kv_heads, d=d, sequences=7, positions=6 * size + 5, dtype=dtype)
    host = HostCache(cache)
    refused = 0
    for step in range(150):
        op = r.choice(["append", "append", "append", "trim", "fork", "compact"])
        some = r.sample(range(7), r.randint(1, 5))
        if op == "append":
            counts = [r.choice([0, 1, 2, size - 1, size, size + 1, 2 * size]) for _ in some]
            held = sum(counts) + 3
            k, v, hk, hv = new_rows(cache, held, step)
            rows = sorted(r.sample(range(held), sum(counts)))
            cache.append(ints(some), starts_of(counts), k, v, ints(rows))
            ok = host.append(some, counts, hk, hv, rows) or sum(counts) == 0
        elif op == "trim":
            lens = [r.choice([0, 0, max(0, int(host.lens[s]) - r.randint(0, size)), int(host.lens[s]) // size * size, 10 ** 6])
                    for s in some]
            cache.trim(ints(some), ints(lens))
            ok = host.trim(some, lens)
        elif op == "fork":
            children = [s for s in range(7) if host.lens[s] == 0 and (host.tables[s] == -1).all()][:3]
            parents = [s for s in range(7) if s not in children]
            if not children or not parents:
                continue
            parents = [r.choice(parents) for _ in children]
            cache.fork(ints(parents), ints(children))
            ok = host.fork(parents, children)
        else:
            cache.compact()
            ok = host.compact()
        host.same(cache)
        status = cache.status()
        assert (status == 0) == ok, (op, status, ok)
        refused += not ok
    assert refused > 0


def test_rows_in_order_and_by_layer():
    """Without a row list token t is row t; extend and write by layer give what append gives."""
    a, b = new_cache(), new_cache()
    counts = [17, 0, 31]
    k, v, hk, hv = new_rows(a, 48, 3)
    host = HostCache(a)
    a.append(ints([4, 1, 6]), starts_of(counts), k, v)
    assert host.append([4, 1, 6], counts, hk, hv, range(48))
    host.same(a)
    b.extend(ints([4, 1, 6]), starts_of(counts))
    for layer in range(b.layers):
        b.write(layer, ints([4, 1, 6]), starts_of(counts), k[layer], v[layer])
    host.same(b)


def test_strided_rows():
    """Keys and values as slices of a fused projection of every layer."""
    cache = new_cache()
    host = HostCache(cache)
    fused = torch.randn(cache.layers, 20, 7, cache.head_dim, device="cuda").to(cache.dtype)
    k, v = fused[:, :, 3:5], fused[:, :, 5:7]
    cache.append(ints([2]), ints([0, 20]), k, v)
    assert host.append([2], [20], *(t.contiguous().cpu().view(torch.int16).numpy() for t in (k, v)), range(20))
    host.same(cache)


def test_no_sequences_and_no_tokens():
    cache = new_cache()
    host = HostCache(cache)
    none, k = ints([]), torch.zeros(2, 0, 2, 64, dtype=torch.bfloat16, device="cuda")
    cache.append(none, ints([0]), k, k)
    cache.trim(none, none)
    cache.fork(none, none)
    cache.compact()
    cache.append(ints([1]), ints([0, 0]), k, k)
    host.same(cache)
    assert cache.status() == 0


def test_forks_are_independent_and_share_full_pages():
    cache = new_cache()
    host = HostCache(cache)
    k, v, hk, hv = new_rows(cache, 37, 5)
    cache.append(ints([0]), ints([0, 37]), k, v)
    host.append([0], [37], hk, hv, range(37))
    cache.fork(ints([0, 0, 0]), ints([3, 1, 7]))
    host.fork([0, 0, 0], [3, 1, 7])
    host.same(cache)
    assert cache.refs.max().item() == 4 and int((cache.refs > 0).sum()) == 2 + 4
    cache.append(ints([1, 0]), ints([0, 3, 8]), k, v)
    host.append([1, 0], [3, 5], hk, hv, range(8))
    cache.trim(ints([0, 3]), ints([0, 0]))
    host.trim([0, 3], [0, 0])
    cache.compact()
    host.compact()
    host.same(cache)
    assert cache.status() == 0


def test_refusals_change_nothing():
    cache = new_cache(pages=5)
    k, v, hk, hv = new_rows(cache, 400, 1)
    cache.append(ints([0, 1]), ints([0, 32, 40]), k, v)
    cache.fork(ints([0]), ints([2]))
    host = HostCache(cache)
    assert cache.status() == 0

    def refused(bit, what):
        what()
        assert cache.status() == bit
        host.same(cache)

    refused(EXHAUSTED, lambda: cache.append(ints([3]), ints([0, 33]), k, v))           # the pool is short of a page
    refused(EXHAUSTED, lambda: cache.append(ints([3]), ints([0, 300]), k, v))          # longer than a table
    refused(BAD_SEQUENCE, lambda: cache.append(ints([3, 3]), ints([0, 1, 2]), k, v))   # named twice
    refused(BAD_SEQUENCE, lambda: cache.append(ints([8]), ints([0, 1]), k, v))
    refused(BAD_SEQUENCE, lambda: cache.append(ints([-1]), ints([0, 1]), k, v))
    refused(BAD_SEQUENCE, lambda: cache.append(ints([3, 4]), ints([0, 5, 3]), k, v))   # a negative count
    refused(SHARED_CUT, lambda: cache.trim(ints([0]), ints([20])))
    refused(BAD_SEQUENCE, lambda: cache.trim(ints([0, 0]), ints([0, 0])))
    refused(BAD_SEQUENCE, lambda: cache.trim(ints([0]), ints([-4])))
    refused(BAD_SEQUENCE, lambda: cache.fork(ints([0]), ints([1])))                    # a child in use
    refused(BAD_SEQUENCE, lambda: cache.fork(ints([3, 0]), ints([4, 3])))              # a child that is a parent
    refused(BAD_SEQUENCE, lambda: cache.fork(ints([9]), ints([4])))
    refused(BAD_SEQUENCE, lambda: cache.fork(ints([0, 1]), ints([4, 4])))
    cache.append(ints([3]), ints([0, 20]), k, v)                                        # the last two pages
    host = HostCache(cache)
    refused(EXHAUSTED, lambda: cache.fork(ints([1]), ints([4])))


def test_rows_out_of_range_are_reported_and_not_written():
    cache = new_cache()
    k, v, hk, hv = new_rows(cache, 4, 1)
    host = HostCache(cache)
    cache.append(ints([0]), ints([0, 3]), k, v, ints([0, 9, 2]))
    assert cache.status() == BAD_INDEX
    page = int(cache.tables[0, 0])
    for slot, row in ((0, 0), (2, 2)):
        host.k[:, page, :, slot], host.v[:, page, :, slot] = hk[:, row], hv[:, row]
    assert np.array_equal(cache.k.cpu().view(torch.int16).numpy(), host.k)


def test_large_pool():
    """More pages than the planning block has threads, most of them taken."""
    cache = new_cache(layers=1, pages=5000, size=16, kv_heads=1, sequences=100, positions=1000)
    r = np.random.RandomState(0)
    host = HostCache(cache)
    lens = r.randint(1, 900, 100)
    pages = iter(r.permutation(5000))
    for s, n in enumerate(lens):
        for p in range(-(-int(n) // 16)):
            host.tables[s, p] = next(pages)
            host.refs[host.tables[s, p]] = 1
    host.lens[:] = lens
    for name in ("tables", "lens", "refs"):
        getattr(cache, name).copy_(torch.from_numpy(getattr(host, name)))
    counts = [int(x) for x in r.randint(0, 40, 100)]
    k, v, hk, hv = new_rows(cache, sum(counts), 7)
    cache.append(ints(range(100)), starts_of(counts), k, v)
    assert host.append(range(100), counts, hk, hv, range(sum(counts)))
    gone = [int(s) for s in r.permutation(100)[:30]]
    cache.trim(ints(gone), ints([0] * 30))
    host.trim(gone, [0] * 30)
    host.same(cache)
    left = [s for s in range(100) if s not in gone]
    cache.fork(ints(left[:30]), ints(gone))
    host.fork(left[:30], gone)
    cache.compact()
    host.compact()
    host.same(cache)
    assert cache.status() == 0


def test_python_argument_checks():
    cache = new_cache()
    k, v, _, _ = new_rows(cache, 4, 1)
    with pytest.raises(ValueError):
        cache.append(ints([0]).long(), ints([0, 4]), k, v)
    with pytest.raises(ValueError):
        cache.append(ints([0]), ints([0]), k, v)
    with pytest.raises(ValueError):
        cache.append(ints([0]), ints([0, 4]), k.half(), v.half())
    with pytest.raises(ValueError):
        cache.append(ints([0]), ints([0, 4]), k[:1], v[:1])
    with pytest.raises(ValueError):
        cache.trim(ints([0]), ints([0, 1]))
    with pytest.raises(ValueError):
        cache.fork(ints([0]).cpu(), ints([1]).cpu())


def test_status_waits_for_every_stream():
    cache = new_cache()
    sequences, lens = ints([cache.tables.shape[0]]), ints([0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)  # about 10 ms, which a status read on another stream would not wait for
    cache.trim(sequences, lens, stream=side)
    assert cache.status() == BAD_SEQUENCE
    assert cache.status() == 0
