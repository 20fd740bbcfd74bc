"""8-bit rows against the definitions in 64 bits: plain, gated and normalised ones."""

import pytest
import torch

from tests._fp8 import check_rows, scales_of, spread
from xpu_playground_b200 import kernels as K

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16
SHAPES = [(1, 16), (1, 128), (3, 112), (5, 144), (2, 1024), (7, 4096), (1, 12288), (129, 2064), (1000, 48), (300, 4096)]


def randn(seed, rows, width, dtype, size=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, width, generator=g) * size
    x[:, ::37] *= 30
    return x.to(dtype)


def silu(x):
    return x * torch.sigmoid(x)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("rows,width", SHAPES)
def test_quantize(rows, width, dtype):
    x = randn(1, rows, width, dtype)
    q, scales = K.fp8_quantize(x.cuda())
    values = check_rows(q, scales, x.double(), 0.0)
    assert (values.abs().amax(1) > 0).all()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("rows,width", SHAPES)
def test_silu_multiply(rows, width, dtype):
    x = randn(2, rows, 2 * width, dtype, 2.0)
    q, scales = K.fp8_silu_multiply(x.cuda())
    gate, up = x.double().chunk(2, 1)
    check_rows(q, scales, silu(gate) * up, 2.0 ** -16)


# Mean of squares: up to 32 additions in a thread and 10 between them, each off by 2^-24; half of that
# in the square root; the root, the quotient and two products behind it.
NORM_OFF = (42 / 2 + 6) * 2.0 ** -24


def norm64(t, weight, epsilon):
    t = t.double()
    return t / torch.sqrt(t.square().mean(1, keepdim=True) + epsilon) * weight.double()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("rows,width", SHAPES + [(2, 8208), (2, 16384), (3, 16400), (2, 32768)])
def test_rms_norm(rows, width, dtype):
    x, r, w = randn(3, rows, width, dtype), randn(4, rows, width, dtype, 4.0), randn(5, 1, width, dtype)[0]
    total, q, scales = K.fp8_rms_norm(x.cuda(), w.cuda(), r.cuda(), 1e-6)
    want = (x.float() + r.float()).to(dtype)
    assert torch.equal(total.cpu(), want)
    check_rows(q, scales, norm64(want, w, 1e-6), NORM_OFF)
    alone, q, scales = K.fp8_rms_norm(x.cuda(), w.cuda(), epsilon=0.5)
    assert torch.equal(alone.cpu(), x)
    check_rows(q, scales, norm64(x, w, 0.5), NORM_OFF)


def test_rows_of_zeros_and_of_the_smallest_numbers():
    x = torch.zeros(4, 256, dtype=BF16)
    x[1, 130] = 2.0 ** -133   # the smallest bf16
    x[2] = 2.0 ** -126
    x[3, 5] = -3.0
    q, scales = K.fp8_quantize(x.cuda())
    check_rows(q, scales, x.double(), 0.0)
    assert (scales[:, 0] == 2.0 ** -126).all() and (q[0].float() == 0).all()
    _, q, scales = K.fp8_rms_norm(x.cuda(), torch.ones(256, dtype=BF16, device="cuda"), epsilon=1e-6)
    check_rows(q, scales, norm64(x, torch.ones(256), 1e-6), NORM_OFF)
    q, scales = K.fp8_silu_multiply(x.cuda())
    check_rows(q, scales, silu(x.double()[:, :128]) * x.double()[:, 128:], 2.0 ** -16)


def test_largest_finite_numbers():
    x = torch.full((2, 128), torch.finfo(BF16).max, dtype=BF16)
    x[1, 3:] = 1e38
    q, scales = K.fp8_quantize(x.cuda())
    check_rows(q, scales, x.double(), 0.0)


@pytest.mark.parametrize("gate", [-1e4, -200.0, -100.0, -88.5, -87.0, -20.0, 0.0, 20.0, 100.0, 6e4])
def test_gates_far_from_zero(gate):
    x = torch.full((1, 256), gate, dtype=BF16)
    x[0, 128:] = torch.linspace(-2, 2, 128).to(BF16)
    q, scales = K.fp8_silu_multiply(x.cuda())
    g, u = x.double().chunk(2, 1)
    y = silu(g) * u
    if scales_of(y).max() > 2.0 ** -100:
        check_rows(q, scales, y, 2.0 ** -16)
    else:  # below what the fast division keeps: nothing is left of them
        assert (q.double().cpu() * spread(scales.double().cpu(), 128)).abs().max() < 2.0 ** -100


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_is_not_finite_stays_so(bad):
    x = randn(6, 4, 384, BF16)
    x[2, 200] = bad
    q, scales = K.fp8_quantize(x.cuda())
    values = q.double().cpu() * spread(scales.double().cpu(), 384)
    assert not torch.isfinite(values[2, 200])
    rest = torch.ones(4, 384, dtype=torch.bool)
    rest[2, 128:256] = False  # its group
    assert torch.isfinite(values[rest]).all()
    _, q, scales = K.fp8_rms_norm(x.cuda(), torch.ones(384, dtype=BF16, device="cuda"))
    values = q.double().cpu() * spread(scales.double().cpu(), 384)
    assert not torch.isfinite(values[2, 200]) and torch.isfinite(values[[0, 1, 3]]).all()


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_rows_that_stand_apart(dtype):
    x, r, w = randn(7, 9, 400, dtype).cuda(), randn(8, 9, 640, dtype).cuda(), randn(9, 1, 144, dtype)[0].cuda()
    for got, want in [(K.fp8_quantize(x[:, 16:160]), K.fp8_quantize(x[:, 16:160].contiguous())),
                      (K.fp8_silu_multiply(x[:, 8:296]), K.fp8_silu_multiply(x[:, 8:296].contiguous())),
                      (K.fp8_rms_norm(x[:, :144], w, r[:, 64:208]), K.fp8_rms_norm(x[:, :144].contiguous(), w, r[:, 64:208].contiguous()))]:
        for a, b in zip(got, want):
            assert torch.equal(a.float(), b.float())


def test_total_in_place_and_given_outputs():
    x, r, w = (randn(i, 33, 1040, BF16).cuda() for i in (1, 2, 3))
    want = K.fp8_rms_norm(x, w[0].contiguous(), r)
    for place in (r.clone(), x.clone()):
        a, b = (x, place) if torch.equal(place, r) else (place, r)
        q, scales = torch.empty_like(want[1]), torch.empty_like(want[2])
        got = K.fp8_rms_norm(a, w[0].contiguous(), b, total=place, q=q, scales=scales)
        assert got[0] is place and got[1] is q and got[2] is scales
        assert all(torch.equal(p.float(), s.float()) for p, s in zip(got, want))


def test_no_rows():
    x = torch.empty(0, 256, dtype=BF16, device="cuda")
    q, scales = K.fp8_quantize(x)
    assert q.shape == (0, 256) and scales.shape == (2, 0)
    assert K.fp8_silu_multiply(x)[0].shape == (0, 128)
    assert K.fp8_rms_norm(x, torch.ones(256, dtype=BF16, device="cuda"))[1].shape == (0, 256)


def test_rows_repeat_and_memory_behind_them_stays():
    x = randn(11, 50, 4096, FP16).cuda()
    q, scales = torch.zeros(51, 4096, dtype=torch.uint8, device="cuda").view(K.FP8), torch.full((32 * 50 + 8,), 7.0, device="cuda")
    K.fp8_quantize(x, q[:50], scales[:1600].view(32, 50))
    again = K.fp8_quantize(x)
    assert torch.equal(q[:50].float(), again[0].float()) and torch.equal(scales[:1600].view(32, 50), again[1])
    assert (q[50].float() == 0).all() and (scales[1600:] == 7).all()
