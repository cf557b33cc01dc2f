"""Timing cases of the text side's batch operators: the linear over 8-bit weights with
scales for each token and channel, and attention of a batch that shares a long prefix
(prompts, chunks and single tokens over the prefix and caches of their own).

``run`` computes each one from elementary torch operations, or through
``iris_b200.kernels`` where ``own`` is set. Shapes are the released trunk's and its text
side's (20 query / 5 key heads of 128, width 2560, 300 prompt tokens, feed-forward 6848) or
generic.
"""

import functools
import math
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one token through an output projection: latency
        dict(name="i8 one token", op="i8", rows=1, inner=2560, outer=2560, products=1, bias=False, dtype="bf16"),
        # one token of 64 sequences through a wide projection: the weights are read once
        dict(name="i8 step of 64", op="i8", rows=64, inner=8192, outer=32768, products=1, bias=False, dtype="bf16"),
        # a ragged chunk through odd widths
        dict(name="i8 odd widths", op="i8", rows=37, inner=6845, outer=2561, products=1, bias=True, dtype="f16"),
        # one prompt in fp32 into the modulation core's width
        dict(name="i8 one prompt", op="i8", rows=301, inner=2560, outer=15360, products=1, bias=True, dtype="f32"),
        # a batch of prompts into both halves of a gated feed-forward, its rows quantised once
        dict(name="i8 gate and up", op="i8", rows=2400, inner=2560, outer=6848, products=2, bias=False, dtype="bf16"),
        # a 2048^2 image's tokens: compute
        dict(name="i8 long", op="i8", rows=16384, inner=8192, outer=8192, products=1, bias=False, dtype="bf16"),
        # one token of a few sequences behind a short instruction: latency
        dict(name="step short prefix", op="prefix", groups=1, batch=4, tokens=1, prefix=300, keys=64, heads=20, kv_heads=5,
             dim=128, right=0, dtype="bf16", ragged=True),
        # one token of 32 sequences behind an instruction of 2048 tokens
        dict(name="step of 32", op="prefix", groups=1, batch=32, tokens=1, prefix=2048, keys=512, heads=32, kv_heads=8,
             dim=128, right=0, dtype="bf16", ragged=True),
        # one token of 64 sequences behind a long document
        dict(name="step long prefix", op="prefix", groups=1, batch=64, tokens=1, prefix=32768, keys=1024, heads=32,
             kv_heads=8, dim=128, right=0, dtype="bf16", ragged=True),
        # five tokens each of four samples of three prompts of their own, prompts of different lengths
        dict(name="chunks of groups", op="prefix", groups=3, batch=12, tokens=5, prefix=1111, keys=203, heads=24, kv_heads=24,
             dim=64, right=0, dtype="f16", ragged=True),
        # a batch of prompts behind an instruction of 4096 tokens
        dict(name="prompts", op="prefix", groups=1, batch=8, tokens=300, prefix=4096, keys=300, heads=20, kv_heads=5, dim=128,
             right=0, dtype="bf16", ragged=False),
        # two images' 1024 tokens, all of them visible to each other, behind one long context
        dict(name="images long prefix", op="prefix", groups=1, batch=2, tokens=1024, prefix=16384, keys=1024, heads=24,
             kv_heads=24, dim=128, right=-1, dtype="f16", ragged=False),
    ]  # fmt: skip


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    if rng.random() < 0.5:
        rows, inner = _log(rng, 1, 16384), _log(rng, 33, 12000)
        outer = _log(rng, 17, min(40000, 268000000 // inner, 134000000 // rows, int(1.0e12 / (rows * inner))))
        return dict(op="i8", rows=rows, inner=inner, outer=outer, products=rng.choice([1, 1, 2]) if rows < 8000 else 1,
                    bias=rng.random() < 0.5, dtype=rng.choice(["bf16", "f16", "f32"]))  # fmt: skip
    kv = rng.choice([1, 2, 3, 4, 5, 8, 16])
    heads = kv * rng.choice([1, 2, 3, 4, 6, 8] if kv < 16 else [1, 2])
    groups = rng.choice([1, 1, 1, 2, 3])
    batch = groups * _log(rng, 1, 64 // groups)
    rooms = int(8.0e8) // (batch * heads)  # (query, key) pairs of one head and sample
    tokens = rng.choice([1, 1, _log(rng, 1, min(1500, int(math.sqrt(rooms))))])
    prefix = _log(rng, 1, min(40000, rooms // (2 * tokens)))
    keys = tokens + rng.choice([0, _log(rng, 1, max(1, min(3000, rooms // (2 * tokens) - tokens)))])
    return dict(op="prefix", groups=groups, batch=batch, tokens=tokens, prefix=prefix, keys=keys, heads=heads, kv_heads=kv,
                dim=rng.choice([64, 128]), right=rng.choice([0, 0, 0, -1, _log(rng, 1, 300)]), dtype=rng.choice(["bf16", "f16"]),
                ragged=rng.random() < 0.5)  # fmt: skip


def _normal(gen, dtype, *shape):
    return torch.randn(*shape, device="cuda", generator=gen).to(dtype)


def _whole(gen, lo, hi, n):
    """n whole numbers of [lo, hi]."""
    return torch.randint(lo, hi + 1, (n,), device="cuda", generator=gen, dtype=torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    c, s = case, {"case": case}
    dt = DTYPES[c["dtype"]]
    if c["op"] == "i8":
        m, k, n = c["rows"], c["inner"], c["outer"]
        # activations whose channels differ in size, a few of them much larger than the others
        size = torch.exp(torch.randn(k, device="cuda", generator=gen))
        s["x"] = (torch.randn(m, k, device="cuda", generator=gen) * size).to(dt)
        s["weights"] = []
        for _ in range(c["products"]):
            w = torch.randn(n, k, device="cuda", generator=gen) * 0.02
            scale = w.abs().amax(dim=1) / 127
            packed = torch.zeros(n, (k + 15) // 16 * 16, device="cuda", dtype=torch.int8)  # rows at 16 bytes
            packed[:, :k] = (w / scale[:, None]).round().clamp(-127, 127).to(torch.int8)
            bias = torch.randn(n, device="cuda", generator=gen) if c["bias"] else None
            s["weights"].append((packed[:, :k], scale, bias))
    else:
        b, n, h, kv, d = c["batch"], c["tokens"], c["heads"], c["kv_heads"], c["dim"]
        # q is read from the packed projection, the caches hold the sequences' own keys
        s["q"] = _normal(gen, dt, b, n, (h + 2 * kv) * d).view(b, n, h + 2 * kv, d).transpose(1, 2)[:, :h]
        s["prefix_k"], s["prefix_v"] = (_normal(gen, dt, c["groups"], kv, c["prefix"], d) for _ in range(2))
        s["k"], s["v"] = (_normal(gen, dt, b, kv, c["keys"], d) for _ in range(2))
        least = n if c["ragged"] else c["keys"]
        s["lengths"] = _whole(gen, least, c["keys"], b)
        s["starts"] = s["lengths"] - n  # the new tokens end each sequence
        s["prefix_lengths"] = None
        if c["groups"] > 1:
            s["prefix_lengths"] = _whole(gen, (c["prefix"] + 1) // 2 if c["ragged"] else c["prefix"], c["prefix"], c["groups"])
    return s


def _limit(n):
    """-1 stands for no bound."""
    return None if n < 0 else n


@functools.cache
def _kernels():
    sys.path.insert(0, "iris-3b-metal_b200")
    from iris_b200 import kernels

    return kernels


def run(s):
    c = s["case"]
    if own:
        K = _kernels()
        if c["op"] == "i8":
            if c["products"] == 1:
                return K.gemm_i8(s["x"], *s["weights"][0])
            q, scale = K.quantize_i8(s["x"])
            return [K.gemm_i8(q, *w, x_scale=scale, out_dtype=s["x"].dtype) for w in s["weights"]]
        return K.prefix_attention(s["q"], s["prefix_k"], s["prefix_v"], s["k"], s["v"], prefix_lengths=s["prefix_lengths"],
                                  starts=s["starts"], lengths=s["lengths"], right=_limit(c["right"]))  # fmt: skip
    if c["op"] == "i8":
        x = s["x"].double()  # which whole number is nearest: 64 bits
        top = x.abs().amax(dim=1, keepdim=True)
        q = (127 * x / torch.where(top == 0, 1.0, top)).round().float()
        out = [_product(q, (top / 127).float(), *w).to(s["x"].dtype) for w in s["weights"]]
        return out[0] if c["products"] == 1 else out
    return _attend(s)


def _product(q, x_scale, packed, scale, bias):
    y = q @ packed.float().T * x_scale * scale
    return y if bias is None else y + bias


def _attend(s):
    """Scores over the group's prefix and the sequence's own keys, one softmax over both."""
    c = s["case"]
    g, b, n, kv, d, h = c["groups"], c["batch"], c["tokens"], c["kv_heads"], c["dim"], c["heads"]
    p, m = c["prefix"], c["keys"]
    q = s["q"].float().reshape(g, b // g, kv, h // kv * n, d)
    by_head = q.transpose(1, 2).reshape(g, kv, -1, d)  # a group's rows of one key head
    early = (by_head @ s["prefix_k"].float().transpose(2, 3)).view(g, kv, b // g, h // kv, n, p)
    late = (q.reshape(b, kv, -1, d) @ s["k"].float().transpose(2, 3)).view(g, b // g, kv, h // kv, n, m).transpose(1, 2)
    z = torch.cat([early, late], dim=-1).mul_(d**-0.5)
    at = s["starts"].long()[:, None, None] + torch.arange(n, device="cuda")[:, None]
    j = torch.arange(m, device="cuda")
    seen = (j < s["lengths"].long()[:, None, None]).expand(b, n, m)
    if c["right"] >= 0:
        seen = seen & (j <= at + c["right"])
    z[..., p:].masked_fill_(~seen.view(g, 1, b // g, 1, n, m), -math.inf)
    if s["prefix_lengths"] is not None:
        hidden = torch.arange(p, device="cuda") >= s["prefix_lengths"].long()[:, None]
        z[..., :p].masked_fill_(hidden.view(g, 1, 1, 1, 1, p), -math.inf)
    top = z.amax(dim=-1, keepdim=True)
    w = z.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = w.sum(dim=-1, keepdim=True)
    out = (w[..., :p].reshape(g, kv, -1, p) @ s["prefix_v"].float()).view(g, kv, b // g, h // kv, n, d)
    own_part = w[..., p:].transpose(1, 2).reshape(b, kv, -1, m) @ s["v"].float()
    out = out + own_part.view(g, b // g, kv, h // kv, n, d).transpose(1, 2)
    out = torch.where(total > 0, out / total, 0.0)
    return out.permute(0, 2, 4, 1, 3, 5).reshape(b, n, h * d).to(s["q"].dtype)


def _own_pairs(c):
    """Visible (query, key) pairs of one head in the sequences' own keys, and such keys, over the batch (lengths at their mean)."""
    n, m = c["tokens"], c["keys"]
    length = (n + m) // 2 if c["ragged"] else m
    if c["right"] < 0:
        return c["batch"] * n * length, c["batch"] * length
    start = length - n
    pairs = sum(min(length, start + i + c["right"] + 1) for i in range(n))
    return c["batch"] * pairs, c["batch"] * min(length, start + n + c["right"])


def work(case):
    c = case
    size = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "i8":
        m, k, n, products = c["rows"], c["inner"], c["outer"], c["products"]
        weights = products * (n * k + 4 * n * (2 if c["bias"] else 1))
        return {"bytes": weights + m * k * size + products * m * n * size, "flops": 2 * products * m * n * k}
    pairs, keys = _own_pairs(c)
    early = 0.75 * c["prefix"] if c["groups"] > 1 and c["ragged"] else c["prefix"]
    rows = 2 * c["batch"] * c["tokens"] * c["heads"] * c["dim"] * size
    return {"bytes": rows + 2 * (c["groups"] * early + keys) * c["kv_heads"] * c["dim"] * size,
            "flops": 4 * (pairs + c["batch"] * c["tokens"] * early) * c["heads"] * c["dim"]}  # fmt: skip


def exact(case, seed):
    """The operators' definitions in 64 bits."""
    c, s = case, prepare(case, seed)
    if c["op"] == "i8":
        out = []
        for packed, scale, bias in s["weights"]:
            y = torch.empty(c["rows"], c["outer"], dtype=torch.float64, device="cuda")
            w = packed.double()
            for i in range(0, c["rows"], 4096):
                x = s["x"][i : i + 4096].double()
                step = x.abs().max(dim=1).values / 127
                levels = torch.div(x, torch.where(step > 0, step, 1.0)[:, None])
                # a quotient this near a half is one: x and step are short numbers
                half = (levels.abs().frac() - 0.5).abs() < 1e-11
                even = 2 * torch.div(levels.abs() + 0.5, 2, rounding_mode="floor") + 0.0
                near = torch.where(half, torch.copysign(even, levels), torch.floor(levels + 0.5))
                y[i : i + 4096] = torch.einsum("mk,nk->mn", near, w) * torch.outer(step, scale.double())
            out.append(y if bias is None else y + bias.double())
        return out[0] if c["products"] == 1 else out
    n, each, per = c["tokens"], c["heads"] // c["kv_heads"], c["batch"] // c["groups"]
    out = torch.zeros(c["batch"], n, c["heads"], c["dim"], dtype=torch.float64, device="cuda")
    first = [c["prefix"]] * c["groups"] if s["prefix_lengths"] is None else s["prefix_lengths"].tolist()
    for b, (start, length) in enumerate(zip(s["starts"].tolist(), s["lengths"].tolist())):
        p = first[b // per]
        own_key = torch.arange(p + length, device="cuda") - p  # below 0: the prefix
        seen = own_key < 0 if c["right"] < 0 else own_key <= start + torch.arange(n, device="cuda")[:, None] + c["right"]
        seen = seen | (own_key < 0) if c["right"] >= 0 else torch.ones(n, p + length, dtype=torch.bool, device="cuda")
        for kv in range(c["kv_heads"]):
            k = torch.cat([s["prefix_k"][b // per, kv, :p], s["k"][b, kv, :length]]).double()
            v = torch.cat([s["prefix_v"][b // per, kv, :p], s["v"][b, kv, :length]]).double()
            z = torch.einsum("hnd,md->hnm", s["q"][b, kv * each : (kv + 1) * each].double(), k) / math.sqrt(c["dim"])
            out[b, :, kv * each : (kv + 1) * each] = torch.softmax(z.masked_fill(~seen, -math.inf), dim=-1).matmul(v).transpose(0, 1)
    return out.flatten(2)
