"""Weights in 8 bits for the products of 8-bit rows (kernels.fp8_gemm)."""

from __future__ import annotations

import torch

from . import kernels
from .kernels import FP8, FP8_BLOCK

LARGEST, SMALLEST_SCALE = 448.0, 2.0 ** -126


class Fp8Weight:
    """A Linear weight [n, k] held as e4m3 with a scale for each block of 128 x
    128: the block's largest value becomes 448. Made once, when a model is
    loaded, without gradients. k is a multiple of 16."""

    @torch.no_grad()
    def __init__(self, weight: torch.Tensor):
        n, k = weight.shape
        if k % 16:
            raise ValueError("the weight's columns must be a multiple of 16")
        blocks = -(-k // FP8_BLOCK)
        self.q = torch.empty(n, k, dtype=FP8, device=weight.device)
        self.scales = torch.empty(-(-n // FP8_BLOCK), blocks, dtype=torch.float32, device=weight.device)
        for begin in range(0, n, 64 * FP8_BLOCK):  # a part at a time: 32 bits of a large weight need room
            rows = weight[begin:begin + 64 * FP8_BLOCK].float()
            at, many = begin // FP8_BLOCK, -(-len(rows) // FP8_BLOCK)
            whole = torch.nn.functional.pad(rows, (0, blocks * FP8_BLOCK - k, 0, many * FP8_BLOCK - len(rows)))
            tiles = whole.view(many, FP8_BLOCK, blocks, FP8_BLOCK)
            scales = (tiles.abs().amax((1, 3)) / LARGEST).clamp(min=SMALLEST_SCALE)
            self.scales[at:at + many] = scales
            q = (tiles / scales[:, None, :, None]).clamp(-LARGEST, LARGEST).to(FP8)
            self.q[begin:begin + len(rows)] = q.view(whole.shape)[:len(rows), :k]

    def __call__(self, rows: tuple[torch.Tensor, torch.Tensor], dtype: torch.dtype = torch.bfloat16, stream=None) -> torch.Tensor:
        """The product of 8-bit rows (q, scales) with the weight, [m, n]."""
        return kernels.fp8_gemm(*rows, self.q, self.scales, dtype=dtype, stream=stream)
