"""Strides of the rows that a cache takes."""

import pytest
import torch

from tests.test_kv_cache_gpu import ints, new_cache, new_rows
from tests.test_kv_write_gpu import content, equal
from xpu_playground_b200._lib import XpuError

pytestmark = pytest.mark.gpu


def bits(*tensors):
    return [t.contiguous().cpu().view(torch.int16) for t in tensors]


def test_rows_that_overlap_are_refused():
    """One row for every position has stride 0: read with a row's length between them, it would run off its memory."""
    cache = new_cache()
    k, v, _, _ = new_rows(cache, 1, 1)
    with pytest.raises(XpuError, match="row stride"):
        cache.append(ints([0]), ints([0, 20]), k.expand(-1, 20, -1, -1), v.expand(-1, 20, -1, -1))
    cache.extend(ints([0]), ints([0, 20]))
    with pytest.raises(XpuError, match="row stride"):
        cache.write(0, ints([0]), ints([0, 20]), k[0].expand(20, -1, -1), v[0].expand(20, -1, -1))
    wide = torch.zeros(1000, dtype=cache.dtype, device="cuda")
    half = wide.as_strided((2, 5, 2, 64), (128, 64, 64, 1))  # rows that begin in the middle of the one before
    with pytest.raises(XpuError, match="row stride"):
        cache.append(ints([1]), ints([0, 5]), half, half)


def test_one_row_and_one_layer_of_any_stride():
    """Where there is one row, or one layer, its stride says nothing."""
    cache = new_cache(layers=1)
    fused = torch.randn(9, 7, 64, device="cuda").to(cache.dtype)
    k, v = fused[:, 3:5], fused[:, 5:7]
    cache.append(ints([0]), ints([0, 9]), k.as_strided((1, 9, 2, 64), (1, 448, 64, 1)), v[None])
    cache.append(ints([1]), ints([0, 1]), k[None, 3:4], v[None, 3:4].clone())
    assert equal(content(cache, 0), bits(k[None], v[None])) and equal(content(cache, 1), bits(k[None, 3:4], v[None, 3:4]))
    two = new_cache(layers=2)
    fused = torch.randn(2, 5, 7, 64, device="cuda").to(two.dtype)
    k, v = fused[:, 2:3, 3:5], fused[:, 2:3, 5:7]
    two.append(ints([3]), ints([0, 1]), k, v)
    assert equal(content(two, 3), bits(k, v)) and two.status() == 0


def test_layers_of_one_stride_zero():
    """The same rows for every layer."""
    cache = new_cache(layers=2)
    k, v, _, _ = new_rows(cache, 6, 1)
    cache.append(ints([0]), ints([0, 6]), k[:1].expand(2, -1, -1, -1), v[:1].expand(2, -1, -1, -1))
    assert equal(content(cache, 0), bits(k[:1].expand(2, -1, -1, -1), v[:1].expand(2, -1, -1, -1)))


def test_layouts_that_differ_are_refused():
    cache = new_cache(layers=2)
    fused = torch.randn(2, 5, 7, 64, device="cuda").to(cache.dtype)
    with pytest.raises(ValueError, match="one layout"):
        cache.append(ints([0]), ints([0, 5]), fused[:, :, :2], fused[:, :, 2:4].contiguous())
