"""Products of 8-bit rows against the definition in 64 bits."""

import pytest
import torch

from tests._fp8 import check_product, product
from xpu_playground_b200 import kernels as K

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def operands(m, n, k, seed=0, spread=3.0):
    """Values over the whole range of e4m3 with scales of many sizes."""
    g = torch.Generator().manual_seed(seed)
    a, w = ((torch.randn(r, k, generator=g) * 60).clamp(-448, 448).to(K.FP8).cuda() for r in (m, n))
    blocks = -(-k // 128)
    a_scales = torch.exp(spread * torch.randn(blocks, m, generator=g)).cuda()
    w_scales = torch.exp(spread * torch.randn(-(-n // 128), blocks, generator=g)).cuda() * 1e-4
    return a, a_scales, w, w_scales


def check(m, n, k, dtype, seed=0, spread=3.0):
    args = operands(m, n, k, seed, spread if dtype == BF16 else min(spread, 1.0))  # inside fp16's range
    if dtype == FP16:
        args[3].mul_(1e-2)
    c = K.fp8_gemm(*args, dtype=dtype)
    want, size = product(*args)
    check_product(c, want, size, k)
    return args, c


SHAPES = [(1, 1, 16), (1, 16, 16), (1, 128, 128), (2, 129, 144), (3, 7, 272), (1, 6144, 1024), (5, 1000, 4096), (16, 384, 4096),
          (17, 130, 2064), (31, 256, 128), (33, 640, 1024), (64, 1024, 512), (65, 513, 768), (127, 128, 400), (128, 256, 4096),
          (129, 255, 1040), (200, 2048, 256), (255, 1, 128), (256, 257, 272), (257, 512, 1024), (300, 1280, 2048), (511, 200, 640),
          (777, 384, 1536), (1025, 300, 144), (2048, 640, 512), (1, 4096, 12288), (40, 128, 12288)]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product(m, n, k, dtype):
    check(m, n, k, dtype, seed=m + n + k)


def test_scales_of_one_size():
    check(100, 300, 1024, BF16, spread=0.0)


def test_largest_values():
    a = torch.full((3, 256), 448.0).to(K.FP8).cuda()
    w = torch.full((5, 256), -448.0).to(K.FP8).cuda()
    ones = torch.ones(2, 3, device="cuda"), torch.ones(1, 2, device="cuda")
    c = K.fp8_gemm(a, ones[0], w, ones[1])
    check_product(c, *product(a, ones[0], w, ones[1]), 256)


def test_a_bad_row_stays_alone():
    """NaN and infinite scales reach their own row, or their own 128 columns, and no other."""
    a, a_scales, w, w_scales = operands(70, 300, 400, 3, 0.0)
    want = K.fp8_gemm(a, a_scales, w, w_scales)
    a_scales[1, 5] = float("nan")
    a.view(torch.uint8)[69, 17] = 0x7F
    w_scales[2, 3] = float("inf")
    got = K.fp8_gemm(a, a_scales, w, w_scales)
    bad = torch.zeros(70, 300, dtype=torch.bool, device="cuda")
    bad[5], bad[69], bad[:, 256:] = True, True, True
    assert not torch.isfinite(got[bad]).any() and torch.equal(got[~bad], want[~bad])


@pytest.mark.parametrize("m,n,k", [(3, 200, 1024), (130, 200, 1024), (600, 777, 256)])
def test_products_repeat_and_memory_behind_them_stays(m, n, k):
    args = operands(m, n, k, 5)
    held = torch.full((m * n + 64,), 7.0, dtype=BF16, device="cuda")
    out = held[:m * n].view(m, n)
    assert K.fp8_gemm(*args, out=out) is out
    for _ in range(3):
        assert torch.equal(K.fp8_gemm(*args), out)
    assert (held[m * n:] == 7).all()


def test_rows_do_not_depend_on_their_number():
    """Each row's sums are its own, whatever stands beside it, within the bounds of the arithmetic."""
    a, a_scales, w, w_scales = operands(300, 256, 1024, 6)
    want, size = product(a, a_scales, w, w_scales)
    for m in (1, 16, 100, 299):
        check_product(K.fp8_gemm(a[:m], a_scales[:, :m].contiguous(), w, w_scales), want[:m], size[:m], 1024)


def test_no_rows():
    a, a_scales, w, w_scales = operands(2, 256, 256)
    assert K.fp8_gemm(a[:0], a_scales[:, :0], w, w_scales).shape == (0, 256)


def test_device_status_is_clean():
    K.device_status()
    check(513, 1000, 1024, BF16)
    check(4, 1000, 4096, BF16)
    assert K.device_status() == 0
