"""Plain 64-bit restatements of the 8-bit rows, their products and sampling, for their tests."""

from __future__ import annotations

import numpy as np
import torch

HALF_STEP, SMALLEST_HALF = 2.0 ** -4, 2.0 ** -10  # of e4m3: relative to a normal value; of the subnormal ones


def scales_of(y):
    """Scales [blocks, rows] of rows y in 64 bits."""
    parts = [p.abs().amax(1) / 448.0 for p in y.split(128, 1)]
    return torch.stack(parts).clamp(min=2.0 ** -126)


def spread(scales, width):
    """[blocks, rows] -> [rows, width]"""
    return scales.t().repeat_interleave(128, 1)[:, :width]


def check_rows(q, scales, y, off):
    """Rows q with `scales` against y, known to a relative error of `off` of FP32 arithmetic: the scale is off by as
    much (and one rounding of the quotient); a value by half a step of e4m3 and as much again."""
    q, scales, want = q.double().cpu(), scales.double().cpu(), scales_of(y)
    off = off + 2.0 ** -22  # roundings of the quotient, the reciprocal and the product with it
    assert torch.isfinite(q).all() and torch.isfinite(scales).all()
    assert ((scales - want).abs() <= off * want).all()
    s = spread(want, y.shape[1])
    bound = torch.maximum((HALF_STEP + 2 * off) * y.abs(), SMALLEST_HALF * (1 + 2 * off) * s) + 2 * off * y.abs()
    assert ((q * spread(scales, y.shape[1]) - y).abs() <= bound).all()
    return q


def product(a, a_scales, w, w_scales):
    """The product in 64 bits, and the sum of its terms' magnitudes."""
    a = a.double().cpu() * spread(a_scales.double().cpu(), a.shape[1])
    n, k = w.shape
    w = w.double().cpu() * w_scales.double().cpu().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    return a @ w.t(), a.abs() @ w.abs().t()


def check_product(c, want, size, k):
    """One rounding to the output's type. In FP32: the 128 products of a group are exact and each of their additions is off by
    at most 2^-23 of the magnitudes (the tensor cores cut off instead of rounding); the scales' product, its use and the sum
    over the groups are k / 128 + 2 roundings."""
    unit = torch.finfo(c.dtype).eps / 2
    tiny = torch.finfo(c.dtype).smallest_normal * torch.finfo(c.dtype).eps  # a step of the subnormal numbers
    off = (128 + k / 128 + 2) * 2.0 ** -23 * size
    bad = (c.double().cpu() - want).abs() > unit * want.abs() + (1 + unit) * off + tiny
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} products out of bounds"


def choose(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Token and logarithm of its probability for one row, by sorting it in 64 bits."""
    x = np.asarray(logits, np.float64)
    settings = (u, temperature, top_p, min_p)
    if (np.isnan(x).any() or np.isposinf(x).any() or np.isneginf(x).all() or any(np.isnan(settings)) or temperature < 0 or
            top_k < 0 or not 0 <= u < 1):
        return -1, -np.inf
    order = np.argsort(-x, kind="stable")
    order = order[~np.isneginf(x[order])]
    if temperature == 0:
        return int(order[0]), 0.0
    with np.errstate(over="ignore"):
        z = (x[order] - x[order[0]]) / np.float64(temperature)
    if top_k:
        z = z[:top_k]
    w = np.exp(z)
    sums = np.cumsum(w)
    keep = max(1, min(int((np.concatenate([[0.0], sums[:-1]]) < np.float64(top_p) * sums[-1]).sum()), int((w >= min_p).sum())))
    at = min(int((sums[:keep] <= np.float64(u) * sums[keep - 1]).sum()), keep - 1)
    return int(order[at]), float(z[at] - np.log(sums[keep - 1]))
