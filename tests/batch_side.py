"""Plain forms in 64 bits of the text side's batch operators, with the error that each
kernel's roundings allow, element by element (shared by the CPU and GPU tests)."""

import math

import torch

from text_side import HALF_STEP, SUBNORMAL


def quantized(x):
    """(whole numbers as fp64 [M, K], FP32 scales [M]) of the rows of x."""
    a = x.double()
    top = a.abs().amax(dim=1) if x.shape[1] else a.new_zeros(x.shape[0])
    fine = torch.isfinite(a).all(dim=1)
    top = torch.where(fine, top, 0.0)
    # 127 x is exact, and a quotient of two short numbers that is no half is further from one than fp64's rounding
    q = (127 * torch.where(fine[:, None], a, 0.0) / torch.where(top == 0, 1.0, top)[:, None]).round()
    scale = top.float() / torch.tensor(127.0, device=x.device)
    return q, torch.where(fine, scale, math.nan)


def assert_i8(got, q, x_scale, packed, scale, bias=None):
    """The sum is exact; its conversion, two products and an addition round to fp32, and the result to its type."""
    exact = (q.double() @ packed.double().T) * x_scale.double()[:, None] * scale.double()
    size = exact.abs()
    if bias is not None:
        exact, size = exact + bias.double(), size + bias.double().abs()
    fine = torch.isfinite(x_scale)[:, None] & torch.isfinite(scale)
    assert bool(torch.isnan(got[~fine.expand_as(got)]).all())
    # the smallest fp32 steps: a product below 2^-126 keeps 2^-149
    off = 4 * 2.0**-24 * size + 2.0**-148
    allowed = off * (1 + HALF_STEP[got.dtype]) + HALF_STEP[got.dtype] * exact.abs() + SUBNORMAL[got.dtype]
    assert torch.all(((got.double() - exact).abs() <= allowed) | ~fine)
