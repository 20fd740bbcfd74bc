"""Rows that the kernel right before has written: calls that follow each other with nothing in between."""

import pytest
import torch

from tests.test_kv_cache_gpu import ints, new_cache
from tests.test_kv_write_gpu import content, equal
from tests.test_serving_attention_gpu import randn
from xpu_playground_b200 import kernels as K

pytestmark = pytest.mark.gpu


def test_rows_of_the_kernel_before():
    """A matrix-vector product into the rows, then the append, again and again into the same rows."""
    cache = new_cache(layers=1, pages=200, kv_heads=2, sequences=40, positions=80)
    m = 64 * 2 * 64
    matrices, vectors = [randn(i, m, 256) for i in range(4)], [randn(10 + i, 256) for i in range(40)]
    rows = torch.zeros(m, dtype=cache.dtype, device="cuda")
    view, starts = rows.view(1, 64, 2, 64), ints([0, 64])
    ids = [ints([i]) for i in range(40)]
    torch.cuda.synchronize()
    for i in range(40):
        K.gemv(matrices[i % 4], vectors[i], out=rows)
        cache.append(ids[i], starts, view, view)
    assert cache.status() == 0
    for i in range(40):
        want = K.gemv(matrices[i % 4], vectors[i]).view(1, 64, 2, 64).cpu().view(torch.int16)
        assert equal(content(cache, i), [want, want])
