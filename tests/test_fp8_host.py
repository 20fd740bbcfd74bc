"""Refusals of the 8-bit operators and of sampling, without a GPU: no work is queued for them."""

import pytest
import torch

from xpu_playground_b200 import _lib
from xpu_playground_b200 import kernels as K

INVALID, UNSUPPORTED = _lib.XPU_ERR_INVALID, _lib.XPU_ERR_UNSUPPORTED

ROWS = dict(dtype=0, x=64, stride=256, q=64, scales=64, rows=3, width=256)
GATED = dict(dtype=0, gate=64, up=576, stride=512, q=64, scales=64, rows=3, width=256)
NORM = dict(dtype=1, x=64, x_stride=256, residual=64, residual_stride=256, weight=64, epsilon=1e-6, total=64, total_stride=256, q=64,
            scales=64, rows=3, width=256)
GEMM = dict(dtype=0, a=64, a_scales=64, w=64, w_scales=64, c=64, m=4, n=5, k=256)
SAMPLE = dict(dtype=0, logits=64, stride=1000, temperature=64, top_k=64, top_p=64, min_p=64, u=64, tokens=64, logprobs=64, rows=3,
              vocabulary=1000)


def refused(name, args, change, status):
    assert getattr(_lib.load(), name)(*(args | change).values(), None) == status
    assert name in _lib.last_error()


@pytest.mark.parametrize("change", [{"x": None}, {"q": None}, {"scales": None}, {"x": 72}, {"q": 68}, {"scales": 66}, {"dtype": 2}, {"width": 0},
                                    {"width": 250}, {"width": 264}, {"stride": 248}, {"stride": 260}, {"stride": 1 << 32},
                                    {"rows": 1 << 31}])
def test_quantize(change):
    refused("xpu_fp8_quantize", ROWS, change, INVALID)


@pytest.mark.parametrize("change", [{"gate": None}, {"up": None}, {"up": 580}, {"gate": 8}, {"q": None}, {"scales": None}, {"dtype": -1},
                                    {"width": 136}, {"stride": 255}, {"stride": 8}])
def test_silu_multiply(change):
    refused("xpu_fp8_silu_multiply", GATED, change, INVALID)


@pytest.mark.parametrize("change", [{"x": None}, {"weight": None}, {"q": None}, {"scales": None}, {"weight": 66}, {"residual": 72},
                                    {"total": 72}, {"residual_stride": 128}, {"total_stride": 257}, {"x_stride": 0}, {"width": 40},
                                    {"epsilon": -1.0}, {"epsilon": float("nan")}, {"epsilon": float("inf")}, {"dtype": 3}])
def test_rms_norm(change):
    refused("xpu_fp8_rms_norm", NORM, change, INVALID)


def test_rms_norm_too_wide():
    wide = dict.fromkeys(("width", "x_stride", "residual_stride", "total_stride"), 32784)
    refused("xpu_fp8_rms_norm", NORM, wide, UNSUPPORTED)


@pytest.mark.parametrize("change", [{"a": None}, {"a_scales": None}, {"w": None}, {"w_scales": None}, {"c": None}, {"a": 72}, {"w": 68},
                                    {"c": 66}, {"a_scales": 62}, {"w_scales": 2}, {"dtype": 2}, {"n": 0}, {"k": 0}, {"k": 264},
                                    {"m": 1 << 31}, {"n": 1 << 31}, {"k": 1 << 31}])
def test_gemm(change):
    refused("xpu_fp8_gemm", GEMM, change, INVALID)


@pytest.mark.parametrize("change", [{"logits": None}, {"u": None}, {"tokens": None}, {"logits": 65}, {"u": 66}, {"top_k": 65}, {"tokens": 62},
                                    {"temperature": 1}, {"top_p": 2}, {"min_p": 3}, {"logprobs": 5}, {"stride": 999}, {"stride": 1 << 32},
                                    {"vocabulary": 0}, {"vocabulary": (1 << 20) + 1, "stride": 1 << 21}, {"rows": 1 << 27}, {"dtype": 2}])
def test_sample(change):
    refused("xpu_sample", SAMPLE, change, INVALID)


def test_no_rows_is_nothing_to_do():
    L = _lib.load()
    for name, args, rows in [("xpu_fp8_quantize", ROWS, "rows"), ("xpu_fp8_silu_multiply", GATED, "rows"),
                             ("xpu_fp8_rms_norm", NORM, "rows"), ("xpu_fp8_gemm", GEMM, "m"), ("xpu_sample", SAMPLE, "rows")]:
        assert getattr(L, name)(*(args | {rows: 0}).values(), None) == 0


def bf16(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


def fp8(*shape):
    return torch.zeros(*shape).to(K.FP8)


@pytest.mark.parametrize("call", [
    lambda: K.fp8_quantize(torch.zeros(2, 256)),
    lambda: K.fp8_quantize(bf16(256, 2).t()),
    lambda: K.fp8_quantize(bf16(2, 256), q=fp8(2, 128)),
    lambda: K.fp8_quantize(bf16(2, 256), q=bf16(2, 256)),
    lambda: K.fp8_quantize(bf16(2, 256), scales=torch.zeros(2, 3)),
    lambda: K.fp8_quantize(bf16(2, 256)),
    lambda: K.fp8_quantize(bf16(256)),
    lambda: K.fp8_silu_multiply(bf16(2, 255)),
    lambda: K.fp8_silu_multiply(bf16(2, 512), q=fp8(2, 512)),
    lambda: K.fp8_rms_norm(bf16(2, 256), bf16(128)),
    lambda: K.fp8_rms_norm(bf16(2, 256), torch.zeros(256)),
    lambda: K.fp8_rms_norm(bf16(2, 256), bf16(256), bf16(3, 256)),
    lambda: K.fp8_rms_norm(bf16(2, 256), bf16(256), bf16(2, 256).half()),
    lambda: K.fp8_rms_norm(bf16(2, 256), bf16(256), total=bf16(2, 128)),
    lambda: K.fp8_gemm(fp8(2, 256), torch.zeros(2, 2), fp8(3, 128), torch.zeros(1, 2)),
    lambda: K.fp8_gemm(fp8(2, 256), torch.zeros(2, 3), fp8(3, 256), torch.zeros(1, 2)),
    lambda: K.fp8_gemm(fp8(2, 256), torch.zeros(2, 2), fp8(3, 256), torch.zeros(2, 2)),
    lambda: K.fp8_gemm(bf16(2, 256), torch.zeros(2, 2), fp8(3, 256), torch.zeros(1, 2)),
    lambda: K.fp8_gemm(fp8(2, 256), torch.zeros(2, 2).double(), fp8(3, 256), torch.zeros(1, 2)),
    lambda: K.fp8_gemm(fp8(2, 256), torch.zeros(2, 2), fp8(3, 256), torch.zeros(1, 2), out=bf16(2, 4)),
    lambda: K.fp8_gemm(fp8(2, 256), torch.zeros(2, 2), fp8(3, 512)[:, ::2], torch.zeros(1, 2)),
    lambda: K.sample(torch.zeros(2, 9), torch.zeros(2)),
    lambda: K.sample(bf16(2, 9), torch.zeros(3)),
    lambda: K.sample(bf16(2, 9), torch.zeros(2), top_k=torch.zeros(2)),
    lambda: K.sample(bf16(2, 9), torch.zeros(2), temperature=torch.zeros(1)),
    lambda: K.sample(bf16(2, 9), None),
    lambda: K.sample(bf16(9), torch.zeros(1)),
])
def test_wrappers_refuse(call):
    with pytest.raises(ValueError):
        call()
