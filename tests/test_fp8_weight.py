"""Weights brought to 8 bits, on the host."""

import pytest
import torch

from xpu_playground_b200.fp8 import Fp8Weight
from xpu_playground_b200.kernels import FP8


@pytest.mark.parametrize("n,k", [(1, 16), (128, 128), (129, 144), (300, 400), (8200, 32)])
def test_every_value_is_within_half_a_step(n, k):
    w = torch.randn(n, k, generator=torch.Generator().manual_seed(n)) * torch.logspace(-3, 3, n)[:, None]
    e = Fp8Weight(w)
    assert e.q.dtype == FP8 and e.q.shape == (n, k) and e.scales.shape == (-(-n // 128), -(-k // 128))
    scales = e.scales.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    back = e.q.double() * scales
    # half a step of e4m3, 2^-4 of a value or 2^-10 of the scale, and the roundings of scale and quotient
    assert ((back - w.double()).abs() <= (2.0 ** -4 + 2.0 ** -21) * w.double().abs() + 2.0 ** -10 * (1 + 2.0 ** -20) * scales).all()
    for i in range(0, n, 128):
        for j in range(0, k, 128):
            top = w[i:i + 128, j:j + 128].abs().max()
            assert abs(float(e.scales[i // 128, j // 128]) * 448 / float(top) - 1) <= 2.0 ** -22
            assert float(e.q[i:i + 128, j:j + 128].float().abs().max()) == 448


def test_a_block_of_zeros():
    e = Fp8Weight(torch.zeros(130, 32))
    assert (e.q.float() == 0).all() and (e.scales == 2.0 ** -126).all()


def test_columns_that_cannot_be_loaded_are_refused():
    with pytest.raises(ValueError, match="multiple of 16"):
        Fp8Weight(torch.zeros(16, 24))


def test_a_parameter_leaves_no_graph():
    e = Fp8Weight(torch.nn.Linear(32, 16).weight)
    assert not e.q.requires_grad and not e.scales.requires_grad
