"""Products of many 8-bit rows, which pairs of blocks compute in tiles of 256 x 256 (k_wide in fp8_gemm.cu)."""

import pytest
import torch

from tests._fp8 import check_product, product
from tests._graphs import kernels_of
from tests.test_fp8_gemm_gpu import BF16, FP16, operands
from xpu_playground_b200 import kernels as K

pytestmark = pytest.mark.gpu


def by_pairs(*args, **kwargs):
    names = kernels_of(lambda: K.fp8_gemm(*args, **kwargs))
    assert len(names) == 1 and ("k_wide" in names[0]) != ("k_skinny" in names[0]), names
    return "k_wide" in names[0]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("m,n,k", [(4100, 2056, 1040), (2049, 1999, 1168)])
def test_scales_that_jump_from_group_to_group(m, n, k, dtype):
    """Scales of a group go from one warp to others four groups at a time: those of another group, or of the tile before, would
    be off by a factor of 64 at least. Each pair has one to three tiles of 9 or 10 groups, so that places are used over and over."""
    a, a_scales, w, w_scales = operands(m, n, k, m, 0.0)
    blocks = len(a_scales)
    jump = 8.0 ** torch.tensor([[0, 3, 1, 4, 2][g % 5] for g in range(blocks)], device="cuda")  # neighbours differ
    a_scales *= jump[:, None] * 1e-4 * (1 + torch.arange(m, device="cuda") % 7)
    w_scales *= jump.flip(0)[None, :] * (1 + torch.arange(len(w_scales), device="cuda") % 3)[:, None]
    if dtype == FP16:
        w_scales *= 1e-2
    assert by_pairs(a, a_scales, w, w_scales, dtype=dtype)
    first = K.fp8_gemm(a, a_scales, w, w_scales, dtype=dtype)
    check_product(first, *product(a, a_scales, w, w_scales), k)
    again = torch.empty_like(first)
    for i in range(200):
        if i % 5 == 0:
            K.fp8_quantize(first[:64, :1920].contiguous())  # another kernel before it now and then
        K.fp8_gemm(a, a_scales, w, w_scales, out=again)
        assert torch.equal(again, first)
    assert K.device_status() == 0


def test_calls_of_one_group_one_after_the_other():
    """A pair ends as soon as its only group is done, and another block takes its place: both blocks stay until every arrival of
    the products on their barriers is in."""
    calls = [operands(m, n, k, i, 1.0) for i, (m, n, k) in enumerate([(257, 9999, 16), (777, 4096, 128), (300, 7000, 112), (20, 640, 128)])]
    assert [by_pairs(*x) for x in calls] == [True, True, True, False]
    want = [K.fp8_gemm(*x) for x in calls]
    for x, c in zip(calls, want):
        check_product(c, *product(*x), x[0].shape[1])
    outs = [[torch.empty_like(c) for c in want] for _ in range(8)]
    for _ in range(25):
        for out in outs:
            for x, c in zip(calls, out):
                K.fp8_gemm(*x, out=c)
    torch.cuda.synchronize()
    assert all(torch.equal(c, w) for out in outs for c, w in zip(out, want))
    assert K.device_status() == 0
