"""Reading a cache's status: no bit is lost, and a timeout leaves no trace."""

import pytest
import torch

from tests._serving import HostCache
from tests.test_kv_cache_gpu import ints, new_cache, new_rows
from xpu_playground_b200.kv_cache import BAD_SEQUENCE, TIMEOUT

pytestmark = pytest.mark.gpu


class SlowToClear:
    """A status word whose clearing takes the device about 10 ms."""

    def __init__(self, word):
        self.word, self.device = word, word.device

    def item(self):
        return self.word.item()

    def zero_(self):
        torch.cuda._sleep(20_000_000)
        self.word.zero_()


def test_a_bit_set_on_another_stream_right_after_a_read_is_kept():
    cache = new_cache()
    bad, lens, side = ints([cache.tables.shape[0]]), ints([0]), torch.cuda.Stream()
    cache._status = SlowToClear(cache._status)
    cache.trim(bad, lens)
    assert cache.status() == BAD_SEQUENCE
    cache.trim(bad, lens, stream=side)
    side.synchronize()
    assert cache.status() == BAD_SEQUENCE
    assert cache.status() == 0


def test_a_timeout_is_reported_and_the_cache_is_usable_again():
    """As blocks that gave up leave it: the flag up, tickets half drawn."""
    cache = new_cache()
    host = HostCache(cache)
    cache._status.fill_(TIMEOUT)
    cache._workspace[:8] = ints([1, 3, 0, 2, 1, 1, 0, 0])
    assert cache.status() == TIMEOUT
    assert not cache._workspace.any()
    k, v, hk, hv = new_rows(cache, 20, 1)
    cache.append(ints([0]), ints([0, 20]), k, v)
    host.append([0], [20], hk, hv, range(20))
    host.same(cache)
    assert cache.status() == 0
