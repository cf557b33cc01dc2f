"""Plain forms in 64 bits of the text-side operators, with the error that each
kernel's roundings allow, element by element (shared by the CPU and GPU tests)."""

import math

import torch

HALF_STEP = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
SUBNORMAL = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0**-25}  # half of fp16's smallest step


def turned(x, cos, sin, layout):
    """x [..., N, D] in fp64, its first 2 * cos.shape[-1] columns turned (cos, sin [..., N, R / 2])."""
    r = cos.shape[-1]
    first, second = (slice(0, r), slice(r, 2 * r)) if layout == "half" else (slice(0, 2 * r, 2), slice(1, 2 * r, 2))
    out = x.clone()
    a, b = x[..., first], x[..., second]
    out[..., first], out[..., second] = a * cos - b * sin, a * sin + b * cos
    return out


def assert_turned(got, x, cos, sin, layout):
    """Every element within its rounding: two products and a sum in fp32 (each half
    a step of at most |a| + |b|, times the tables' magnitude), then the row's type."""
    exact = turned(x.double(), cos.double(), sin.double(), layout)
    size = turned(x.double().abs(), cos.double().abs(), -sin.double().abs(), layout).abs()
    size = torch.maximum(size, turned(x.double().abs(), cos.double().abs(), sin.double().abs(), layout).abs())
    r = 2 * cos.shape[-1]
    allowed = HALF_STEP[got.dtype] * exact.abs() + SUBNORMAL[got.dtype]
    allowed[..., :r] += 3 * 2.0**-24 * size[..., :r] * (1 + HALF_STEP[got.dtype])
    assert torch.all((got.double() - exact).abs() <= allowed)


def visible(n, n_kv, starts, lengths, left, right, sinks):
    """bool [B, N, N_kv]."""
    i = starts[:, None, None].long() + torch.arange(n, device=starts.device)[:, None]
    j = torch.arange(n_kv, device=starts.device)
    seen = (j < lengths[:, None, None]).expand(-1, n, -1).clone()
    if right is not None:
        seen &= j <= i + right
    if left is not None:
        seen &= (j >= i - left) | (j < sinks)
    return seen


def attention(q, k, v, seen, scale):
    """fp64 [B, N, H, D] and, per element, what the kernel's roundings allow."""
    b, h, n, d = q.shape
    each = h // k.shape[1]
    out = torch.zeros(b, n, h, d, dtype=torch.float64, device=q.device)
    allowed = torch.zeros_like(out)
    e, tiny = HALF_STEP[q.dtype], SUBNORMAL[q.dtype]
    for s in range(b):
        for head in range(h):
            kk, qq = k[s, head // each].double(), q[s, head].double()
            # what no query of the sample sees takes no part, NaN included
            used = seen[s].any(dim=0)
            kk = torch.where(used[:, None], kk, 0.0)
            vv = torch.where(used[:, None], v[s, head // each].double(), 0.0)
            z = (qq @ kk.T * scale).masked_fill(~seen[s], -math.inf)
            some = seen[s].any(dim=1)[:, None]
            top = torch.where(some, z.amax(dim=1, keepdim=True), 0.0)
            w = torch.where(seen[s], (z - top).exp(), 0.0)
            total = w.sum(dim=1, keepdim=True).clamp_min(1e-300)
            out[s, :, head] = w @ vv / total
            # a score is a sum of d products in fp32, at most 2^-23 of the sum of magnitudes per addition, and its
            # product with the scale, subtraction of the maximum and exponential 2^-21 of it and of one more; it enters
            # numerator and denominator. Each weight is rounded to the type once (fp16 has a smallest step below its
            # largest weight, which is at least 1), the sums to fp32, the result to the type.
            size = ((qq.abs() @ kk.abs().T) * scale).masked_fill(~seen[s], 0).amax(dim=1, keepdim=True)
            score = (d * 2.0**-23 + 2.0**-21) * size + 2.0**-20
            spread = w @ vv.abs() / total
            small = tiny * (seen[s].double() @ vv.abs()) / total
            allowed[s, :, head] = e * out[s, :, head].abs() + (1 + e) * ((e + 2 * score + kk.shape[0] * 2.0**-23) * spread + small) + tiny
    return out, allowed


def assert_attends(got, q, k, v, *, left=None, right=0, sinks=0, starts=None, lengths=None, scale=None):
    b, h, n, d = q.shape
    m = k.shape[2]
    full = torch.full((b,), m, device=q.device)
    starts = full - n if starts is None else starts
    lengths = full if lengths is None else lengths.clamp(0, m)
    seen = visible(n, m, starts, lengths, left, right, sinks)
    exact, allowed = attention(q, k, v, seen, d**-0.5 if scale is None else scale)
    off = (got.double().view(b, n, h, d) - exact).abs()
    assert torch.all(off <= allowed), f"{float((off / allowed.clamp_min(1e-30)).max()):.3g} times what is allowed"


def silu(x):
    return x * torch.sigmoid(x)


def unpacked(packed, scale, zero):
    """fp64 [N, K] of 4-bit weights."""
    n, half = packed.shape
    q = torch.stack([packed % 16, torch.div(packed, 16, rounding_mode="floor")], dim=-1).reshape(n, scale.shape[1], -1).double()
    z = 8.0 if zero is None else zero.double()[..., None]
    return ((q - z) * scale.double()[..., None]).reshape(n, 2 * half)


def assert_q4(got, x, packed, scale, zero, bias, silu_in=False, silu_out=False):
    """fp32 sums: each of the K / 16 accumulations of a chain, the sums over its ends
    and the scales' products off by at most 2^-23 of the sum of magnitudes; a silu in
    fp32 by 2^-18 (its exponent's argument is rounded at up to 16 times 2^-24 log2 e);
    the result is rounded to its type."""
    w = unpacked(packed, scale, zero)
    a = silu(x.double()) if silu_in else x.double()
    exact = a @ w.T + (0 if bias is None else bias.double())
    size = a.abs() @ w.abs().T + (0 if bias is None else bias.double().abs())
    off = (x.shape[1] / 16 + 40) * 2.0**-23 * size + (2.0**-18 * size if silu_in else 0)
    if silu_out:
        off, exact = 1.1 * off + 2.0**-18 * exact.abs(), silu(exact)  # silu's slope is below 1.1
    allowed = off * (1 + HALF_STEP[got.dtype]) + HALF_STEP[got.dtype] * exact.abs() + SUBNORMAL[got.dtype]
    assert torch.all((got.double() - exact).abs() <= allowed)
