"""Plain forms in 64 bits of the text side's batch operators, with the error that each
kernel's roundings allow, element by element (shared by the CPU and GPU tests)."""

import math

import torch

from text_side import HALF_STEP, SUBNORMAL, attention


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


def prefix_seen(n, p, m, prefix_length, start, length, right, device):
    """bool [N, P + M]: the prefix's keys, then the sample's own."""
    own = torch.arange(m, device=device)
    seen = (own < length).expand(n, m).clone()
    if right is not None:
        seen &= own <= start + torch.arange(n, device=device)[:, None] + right
    early = (torch.arange(p, device=device) < prefix_length).expand(n, p)
    return torch.cat([early, seen], dim=1)


def assert_prefix(got, q, pk, pv, k, v, *, prefix_lengths=None, starts=None, lengths=None, right=0, scale=None):
    """Sample by sample over the two lots of keys joined: the sums are the same as in one
    attention over them, in another order, and what the parts' joining rounds (a product and an
    addition in fp32 for each part) is within the sums' allowance."""
    b, h, n, d = q.shape
    p, m, per = pk.shape[2], k.shape[2], b // pk.shape[0]
    worst = 0.0
    for s in range(b):
        first = p if prefix_lengths is None else min(max(int(prefix_lengths[s // per]), 0), p)
        start = m - n if starts is None else int(starts[s])
        length = m if lengths is None else min(max(int(lengths[s]), 0), m)
        seen = prefix_seen(n, p, m, first, start, length, right, q.device)
        keys, values = (torch.cat([a[s // per], e[s]], dim=1)[None] for a, e in ((pk, k), (pv, v)))
        exact, allowed = attention(q[s : s + 1], keys, values, seen[None], d**-0.5 if scale is None else scale)
        off = (got[s].double().view(1, n, h, d) - exact).abs()
        worst = max(worst, float((off / allowed.clamp_min(1e-30)).max()) if off.numel() else 0.0)
        assert torch.all(off <= allowed), f"sample {s}: {worst:.3g} times what is allowed"
    return worst
