"""Rows written layer by layer, with other requests between an extension and its writes."""

import pytest
import torch

from tests.test_kv_cache_gpu import ints, new_cache, new_rows, starts_of
from xpu_playground_b200.kv_cache import BAD_INDEX, BAD_SEQUENCE, EXHAUSTED, SHARED_CUT

pytestmark = pytest.mark.gpu


def content(cache, sequence):
    """Bits of a sequence's rows [layers, length, kv_heads, head_dim], keys and values."""
    n, size = int(cache.lens[sequence]), cache.page_size
    pages = cache.tables[sequence, :-(-n // size)].long()
    return [pool[:, pages].transpose(2, 3).flatten(1, 2)[:, :n].cpu().view(torch.int16) for pool in (cache.k, cache.v)]


def rows_of(k, v, begin, end):
    return [t[:, begin:end].cpu().view(torch.int16) for t in (k, v)]


def equal(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def write_all(cache, sequences, starts, k, v):
    for layer in range(cache.layers):
        cache.write(layer, sequences, starts, k[layer], v[layer])


REFUSED = {
    "fork": (BAD_SEQUENCE, lambda c, k, v: c.fork(ints([0]), ints([1]))),
    "trim": (SHARED_CUT, lambda c, k, v: c.trim(ints([0]), ints([20]))),
    "append": (BAD_SEQUENCE, lambda c, k, v: c.append(ints([5, 5]), ints([0, 1, 2]), k, v)),
}


@pytest.mark.parametrize("what", sorted(REFUSED))
def test_refused_requests_between_the_layers_change_nothing(what):
    cache = new_cache(layers=3)
    k, v, _, _ = new_rows(cache, 60, 1)
    cache.append(ints([0, 1]), ints([0, 32, 40]), k, v)
    cache.fork(ints([0]), ints([2]))
    before = content(cache, 0)
    some, starts = ints([4, 1]), ints([0, 37, 50])
    cache.extend(some, starts)
    bit, request = REFUSED[what]
    for layer in range(3):
        cache.write(layer, some, starts, k[layer], v[layer])
        request(cache, k, v)
    assert cache.status() == bit
    assert equal(content(cache, 4), rows_of(k, v, 0, 37)) and equal(content(cache, 0), before)
    new = [torch.cat([a, b], 1) for a, b in zip(rows_of(k, v, 32, 40), rows_of(k, v, 37, 50))]
    assert equal(content(cache, 1), new)


ACCEPTED = {
    "compact": lambda c, k, v: c.compact(),
    "fork": lambda c, k, v: c.fork(ints([0]), ints([3])),
    "append": lambda c, k, v: c.append(ints([5]), ints([0, 1]), k, v),
    "trim": lambda c, k, v: c.trim(ints([1]), ints([3])),
}


@pytest.mark.parametrize("what", sorted(ACCEPTED))
def test_a_refused_extension_writes_nothing_whatever_is_accepted_behind_it(what):
    cache = new_cache(pages=8)
    k, v, _, _ = new_rows(cache, 200, 1)
    cache.append(ints([0, 1]), ints([0, 48, 60]), k, v)
    some, starts = ints([0]), ints([0, 150])
    cache.extend(some, starts)
    ACCEPTED[what](cache, k, v)
    pools = cache.k.clone(), cache.v.clone()
    write_all(cache, some, starts, k, v)
    assert cache.status() == EXHAUSTED
    assert torch.equal(cache.k.view(torch.int16), pools[0].view(torch.int16))
    assert torch.equal(cache.v.view(torch.int16), pools[1].view(torch.int16))


def test_requests_of_other_sequences_between_an_extension_and_its_writes():
    cache = new_cache(layers=2)
    k, v, _, _ = new_rows(cache, 100, 2)
    cache.append(ints([0, 1, 2]), ints([0, 20, 50, 70]), k, v)
    some, starts = ints([6, 0]), ints([0, 33, 40])
    cache.extend(some, starts)
    cache.trim(ints([1]), ints([0]))
    cache.write(0, some, starts, k[0], v[0])
    cache.fork(ints([2]), ints([3]))
    cache.append(ints([2]), ints([0, 9]), k, v)
    cache.compact()
    cache.write(1, some, starts, k[1], v[1])
    assert cache.status() == 0
    assert equal(content(cache, 6), rows_of(k, v, 0, 33))
    assert equal(content(cache, 0), [torch.cat([a, b], 1) for a, b in zip(rows_of(k, v, 0, 20), rows_of(k, v, 33, 40))])
    assert equal(content(cache, 3), rows_of(k, v, 50, 70))
    assert equal(content(cache, 2), [torch.cat([a, b], 1) for a, b in zip(rows_of(k, v, 50, 70), rows_of(k, v, 0, 9))])


def test_an_extended_sequence_that_changed_keeps_its_other_rows():
    """What was appended to it since stays, what was trimmed off is reported and not written."""
    cache = new_cache(layers=2)
    k, v, _, _ = new_rows(cache, 40, 3)
    cache.append(ints([0, 1]), ints([0, 20, 30]), k, v)
    some, starts = ints([0, 1]), ints([0, 6, 13])
    cache.extend(some, starts)
    cache.append(ints([1]), ints([0, 4]), k, v)
    cache.trim(ints([0]), ints([23]))
    write_all(cache, some, starts, k, v)
    assert cache.status() == BAD_INDEX
    assert equal(content(cache, 0), [torch.cat([a, b], 1) for a, b in zip(rows_of(k, v, 0, 20), rows_of(k, v, 0, 3))])
    parts = [rows_of(k, v, 20, 30), rows_of(k, v, 6, 13), rows_of(k, v, 0, 4)]
    assert equal(content(cache, 1), [torch.cat(p, 1) for p in zip(*parts)])


def test_a_list_that_is_not_the_extensions_is_reported():
    cache = new_cache(layers=1)
    k, v, _, _ = new_rows(cache, 40, 3)
    cache.append(ints([0, 1]), ints([0, 20, 30]), k, v)
    cache.extend(ints([2]), ints([0, 5]))
    before = content(cache, 0), content(cache, 1)
    cache.write(0, ints([0]), ints([0, 5]), k[0], v[0])
    cache.write(0, ints([2, 1]), ints([0, 5, 8]), k[0], v[0])
    assert cache.status() == BAD_INDEX
    assert equal(content(cache, 0), before[0]) and equal(content(cache, 1), before[1])
    assert equal(content(cache, 2), rows_of(k, v, 0, 5))
