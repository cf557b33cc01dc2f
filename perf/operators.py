"""Timing cases of the text-side operators: rotary positions (on their own and
with the append to a key / value cache), attention with a sliding window and
first tokens that stay visible (prompts and single tokens), and the small-M
linear over 4-bit weights.

``run`` computes each one from elementary torch operations in fp32, or through
``iris_b200.kernels`` where ``own`` is set. Shapes are the released trunk's and
its text side's (20 query / 5 key heads of 128, width 2560, 300 prompt tokens, 4096
or 16384 image tokens) or generic.
"""

import functools
import math
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # the heads of a batch of prompts, read in place from the packed projection
        dict(name="rope prompts", op="rope", batch=8, tokens=300, heads=25, dim=128, rotary=128, layout="half",
             dtype="bf16", first=0, inverse=False),
        # a 2048^2 image's tokens: half of each head rotated, far positions, fp32
        dict(name="rope long", op="rope", batch=1, tokens=16384, heads=25, dim=128, rotary=64, layout="interleaved",
             dtype="f32", first=100003, inverse=False),
        # one token of one sequence into a rolling cache that has wrapped many times
        dict(name="append one token", op="append", batch=1, tokens=1, heads=20, kv_heads=5, dim=128, rotary=128,
             layout="half", dtype="bf16", capacity=1028, sinks=4, first=30011, ragged=False),
        # prompts of different lengths, padded to one, into fresh rows of a cache
        dict(name="append prompts", op="append", batch=8, tokens=301, heads=32, kv_heads=8, dim=64, rotary=64,
             layout="interleaved", dtype="f16", capacity=640, sinks=-1, first=37, ragged=True),
        # the causal encoder over a padded batch of prompts
        dict(name="attend prompts", op="attend", batch=4, tokens=300, keys=300, heads=20, kv_heads=5, dim=128, left=-1,
             right=0, sinks=0, dtype="bf16", first=0, ragged=True),
        # a long causal sequence with a window of 1024 and four first tokens
        dict(name="attend long window", op="attend", batch=1, tokens=16384, keys=16384, heads=20, kv_heads=5, dim=128,
             left=1023, right=0, sinks=4, dtype="bf16", first=0, ragged=False),
        # a 1024^2 image's joint sequence: text first and always visible, image tokens near their neighbours
        dict(name="attend text and image", op="attend", batch=2, tokens=4352, keys=4352, heads=24, kv_heads=24, dim=128,
             left=512, right=512, sinks=256, dtype="f16", first=0, ragged=False),
        # one new token over a rolling cache (every slot counts): latency
        dict(name="step rolling cache", op="attend", batch=1, tokens=1, keys=1028, heads=20, kv_heads=5, dim=128,
             left=-1, right=0, sinks=0, dtype="bf16", first=1027, ragged=False),
        # one new token of many sequences over long caches filled to different lengths
        dict(name="step long caches", op="attend", batch=16, tokens=1, keys=32768, heads=32, kv_heads=8, dim=128,
             left=-1, right=0, sinks=0, dtype="bf16", first=32767, ragged=True),
        # the shared modulation core of the released width: six rows of 2560 from one conditioning row
        dict(name="q4 core", op="q4", rows=1, inner=2560, outer=15360, group=64, zeros=False, dtype="f32", silu=True),
        # one token through a wide projection
        dict(name="q4 one token", op="q4", rows=1, inner=8192, outer=32768, group=128, zeros=False, dtype="bf16",
             silu=False),
        # sixteen tokens through a down projection of odd width, weights with zero points
        dict(name="q4 sixteen rows", op="q4", rows=16, inner=6848, outer=2561, group=32, zeros=True, dtype="f16",
             silu=False),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    kv = rng.choice([1, 2, 3, 4, 5, 8])
    return kv * rng.choice([1, 2, 3, 4, 6, 8]), kv


def draw(rng):
    op = rng.choice(["rope", "append", "attend", "step", "q4"])
    if op == "rope":
        dim = rng.choice([64, 80, 128])
        heads, batch = rng.randint(1, 40), rng.randint(1, 8)
        return dict(op="rope", batch=batch, tokens=_log(rng, 1, 400000 // (batch * heads)), heads=heads, dim=dim,
                    rotary=rng.choice([dim, dim // 2]), layout=rng.choice(["half", "interleaved"]),
                    dtype=rng.choice(["bf16", "f16", "f32"]), first=rng.randint(0, 120000),
                    inverse=rng.random() < 0.3)  # fmt: skip
    if op == "append":
        dim = rng.choice([64, 128])
        heads, kv = _heads(rng)
        batch, tokens, rolling = _log(rng, 1, 32), _log(rng, 1, 600), rng.random() < 0.5
        sinks = rng.randint(0, 8) if rolling else -1
        capacity = rng.randint(16, 1500) if rolling else tokens + rng.randint(1, 1000)
        return dict(op="append", batch=batch, tokens=tokens, heads=heads, kv_heads=kv, dim=dim, rotary=dim,
                    layout=rng.choice(["half", "interleaved"]), dtype=rng.choice(["bf16", "f16"]), capacity=capacity,
                    sinks=sinks, first=rng.randint(0, 40000) if rolling else rng.randint(0, capacity - tokens),
                    ragged=rng.random() < 0.5)  # fmt: skip
    if op == "attend":
        heads, kv = _heads(rng)
        batch = rng.randint(1, 4)
        tokens = _log(rng, 2, int(math.sqrt(2e9 / (batch * heads))))
        keys = tokens if rng.random() < 0.7 else tokens + _log(rng, 1, 1000)
        return dict(op="attend", batch=batch, tokens=tokens, keys=keys, heads=heads, kv_heads=kv,
                    dim=rng.choice([64, 128]), left=rng.choice([-1, _log(rng, 1, 4096)]),
                    right=rng.choice([0, 0, -1, _log(rng, 1, 1024)]), sinks=rng.choice([0, 1, 4, _log(rng, 1, 300)]),
                    dtype=rng.choice(["bf16", "f16"]), first=keys - tokens, ragged=rng.random() < 0.5)  # fmt: skip
    if op == "step":
        heads, kv = _heads(rng)
        batch = _log(rng, 1, 32)
        keys = _log(rng, 1, min(40000, 3000000 // (batch * kv)))
        return dict(op="attend", batch=batch, tokens=1, keys=keys, heads=heads, kv_heads=kv,
                    dim=rng.choice([64, 128]), left=rng.choice([-1, -1, _log(rng, 1, 4096)]), right=0,
                    sinks=rng.choice([0, 4]), dtype=rng.choice(["bf16", "f16"]), first=keys - 1,
                    ragged=rng.random() < 0.5)  # fmt: skip
    group = rng.choice([32, 64, 128])
    inner = group * _log(rng, 1, 10000 // group)
    return dict(op="q4", rows=rng.choice([1, 1, 2, 3, 5, 8, 11, 16]), inner=inner,
                outer=_log(rng, 17, min(40000, 268000000 // inner)), group=group, zeros=rng.random() < 0.5,
                dtype=rng.choice(["bf16", "f16", "f32"]), silu=rng.random() < 0.3)  # fmt: skip


def _table(rotary, positions, theta=1000000.0):
    """cos and sin of the angles, evaluated in 64 bits on the GPU and rounded once."""
    freqs = theta ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / rotary)
    angles = torch.outer(torch.arange(positions, dtype=torch.float64, device="cuda"), freqs)
    return angles.cos().float(), angles.sin().float()


def _normal(gen, dtype, *shape):
    return torch.randn(*shape, device="cuda", generator=gen).to(dtype)


def _whole(gen, lo, hi, n):
    """n whole numbers of [lo, hi]."""
    return torch.randint(lo, hi + 1, (n,), device="cuda", generator=gen, dtype=torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    c, s = case, {"case": case}
    dt = DTYPES[c["dtype"]]
    if c["op"] == "rope":
        b, n, h, d = c["batch"], c["tokens"], c["heads"], c["dim"]
        # the packed projection of one layer: the rotated heads, then as many columns of values
        s["x"] = _normal(gen, dt, b, n, 2 * h * d).view(b, n, 2 * h, d)[:, :, :h].transpose(1, 2)
        s["cos"], s["sin"] = _table(c["rotary"], c["first"] + n)
        s["positions"] = torch.arange(c["first"], c["first"] + n, device="cuda")
    elif c["op"] == "append":
        b, n, h, kv, d = c["batch"], c["tokens"], c["heads"], c["kv_heads"], c["dim"]
        qkv = _normal(gen, dt, b, n, (h + 2 * kv) * d).view(b, n, h + 2 * kv, d).transpose(1, 2)
        s["q"], s["k"], s["v"] = qkv[:, :h], qkv[:, h : h + kv], qkv[:, h + kv :]
        s["cos"], s["sin"] = _table(c["rotary"], c["first"] + n)
        s["k_cache"] = _normal(gen, dt, b, kv, c["capacity"], d)
        s["v_cache"] = _normal(gen, dt, b, kv, c["capacity"], d)
        s["starts"] = _whole(gen, c["first"] // 2, c["first"], b) if c["ragged"] else _whole(gen, c["first"], c["first"], b)
        s["counts"] = _whole(gen, 0, n, b) if c["ragged"] else None
    elif c["op"] == "attend":
        b, n, h, kv, d, m = c["batch"], c["tokens"], c["heads"], c["kv_heads"], c["dim"], c["keys"]
        if n == m:  # a prompt: q, k and v read from the packed projection
            qkv = _normal(gen, dt, b, n, (h + 2 * kv) * d).view(b, n, h + 2 * kv, d).transpose(1, 2)
            s["q"], s["k"], s["v"] = qkv[:, :h], qkv[:, h : h + kv], qkv[:, h + kv :]
        else:  # new tokens over a cache
            s["q"] = _normal(gen, dt, b, n, h * d).view(b, n, h, d).transpose(1, 2)
            s["k"], s["v"] = _normal(gen, dt, b, kv, m, d), _normal(gen, dt, b, kv, m, d)
        s["lengths"] = _whole(gen, min(m, n + m // 4), m, b) if c["ragged"] else _whole(gen, m, m, b)
        # the first new token's position: a prompt starts at 0, new tokens end a sequence
        s["starts"] = torch.zeros_like(s["lengths"]) if n == m else s["lengths"] - n
    else:
        n, k, g = c["outer"], c["inner"], c["group"]
        s["x"] = _normal(gen, dt, c["rows"], k)
        s["packed"] = torch.randint(0, 256, (n, k // 2), device="cuda", generator=gen, dtype=torch.uint8)
        s["scale"] = ((0.5 + torch.rand(n, k // g, device="cuda", generator=gen)) * 0.004).to(torch.bfloat16)
        s["zero"] = None
        if c["zeros"]:
            s["zero"] = torch.randint(4, 12, (n, k // g), device="cuda", generator=gen, dtype=torch.uint8)
        s["bias"] = torch.randn(n, device="cuda", generator=gen)
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
        if c["op"] == "rope":
            return K.rope(s["x"], s["cos"], s["sin"], s["positions"], layout=c["layout"], inverse=c["inverse"])
        if c["op"] == "append":
            q = K.rope_append(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["starts"], s["k_cache"], s["v_cache"],
                              sinks=_limit(c["sinks"]), counts=s["counts"], layout=c["layout"])  # fmt: skip
            return q, s["k_cache"], s["v_cache"]
        if c["op"] == "attend":
            return K.window_attention(s["q"], s["k"], s["v"], left=_limit(c["left"]), right=_limit(c["right"]),
                                      sinks=c["sinks"], starts=s["starts"], lengths=s["lengths"])  # fmt: skip
        return K.gemv_q4(s["x"], s["packed"], s["scale"], s["zero"], s["bias"], silu_in=c["silu"])
    if c["op"] == "rope":
        cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]
        return _rotate(s["x"].float(), cos, -sin if c["inverse"] else sin, c["layout"]).to(s["x"].dtype)
    if c["op"] == "append":
        return _append(s)
    if c["op"] == "attend":
        return _attend(s)
    x = s["x"].float()
    x = x / (1 + torch.exp(-x)) if c["silu"] else x
    q = torch.stack([s["packed"] & 15, s["packed"] >> 4], dim=-1).view(c["outer"], -1, c["group"]).float()
    w = (q - (8.0 if s["zero"] is None else s["zero"].float()[..., None])) * s["scale"].float()[..., None]
    return (x @ w.view(c["outer"], c["inner"]).T + s["bias"]).to(s["x"].dtype)


def _rotate(x, cos, sin, layout):
    """The first 2 * cos.shape[-1] columns of x rotated by pairs, the others as they are."""
    r = cos.shape[-1]
    if layout == "half":
        a, b = x[..., :r], x[..., r : 2 * r]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    else:
        a, b = x[..., 0 : 2 * r : 2], x[..., 1 : 2 * r : 2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    return torch.cat([turned, x[..., 2 * r :]], dim=-1)


def _append(s):
    """Each slot of the cache takes the last new token that belongs to it, if there is one."""
    c, n, capacity = s["case"], s["q"].shape[2], s["k_cache"].shape[2]
    first = s["starts"].long()
    count = torch.full_like(first, n) if s["counts"] is None else s["counts"].long()
    at = first[:, None] + torch.arange(n, device="cuda")
    rows = at.clamp_max(s["cos"].shape[0] - 1)
    cos, sin = s["cos"][rows][:, None], s["sin"][rows][:, None]
    real = (torch.arange(n, device="cuda") < count[:, None])[:, None, :, None]
    q = torch.where(real, _rotate(s["q"].float(), cos, sin, c["layout"]), 0.0).to(s["q"].dtype)
    k = _rotate(s["k"].float(), cos, sin, c["layout"]).to(s["k"].dtype)
    slot = torch.arange(capacity, device="cuda").expand(c["batch"], capacity)
    last = (first + count - 1)[:, None]
    p = slot
    if c["sinks"] >= 0:
        turn = last - torch.remainder(last - slot, capacity - c["sinks"])
        p = torch.where(slot < c["sinks"], slot, torch.where(turn >= slot, turn, -1))
    take = ((p >= first[:, None]) & (p <= last))[:, None, :, None]
    token = (p - first[:, None]).clamp(0, n - 1)[:, None, :, None].expand(-1, c["kv_heads"], -1, c["dim"])
    s["k_cache"].copy_(torch.where(take, k.gather(2, token), s["k_cache"]))
    s["v_cache"].copy_(torch.where(take, s["v"].gather(2, token), s["v_cache"]))
    return q, s["k_cache"], s["v_cache"]


def _visible(s):
    """Truth values [B, N, S]: key j for the query at position p."""
    c = s["case"]
    p = (s["starts"].long()[:, None] + torch.arange(c["tokens"], device="cuda"))[..., None]
    j = torch.arange(c["keys"], device="cuda")
    seen = (j < s["lengths"].long()[:, None, None]).expand(-1, c["tokens"], -1)
    seen = seen if c["right"] < 0 else seen & (j <= p + c["right"])
    return seen if c["left"] < 0 else seen & ((j >= p - c["left"]) | (j < c["sinks"]))


def _attend(s):
    c = s["case"]
    b, n, kv, d = c["batch"], c["tokens"], c["kv_heads"], c["dim"]
    q = s["q"].float().reshape(b, kv, -1, d)  # a key head's query heads, one after the other
    scores = (q @ s["k"].float().transpose(2, 3)).mul_(d**-0.5).view(b, kv, c["heads"] // kv, n, c["keys"])
    scores.masked_fill_(~_visible(s)[:, None, None], -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    p = scores.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(dim=-1).view(b, c["heads"], n, 1)
    out = (p.view(b, kv, -1, c["keys"]) @ s["v"].float()).view(b, c["heads"], n, d)
    out = torch.where(total > 0, out / total, 0.0)
    return out.transpose(1, 2).reshape(b, n, c["heads"] * d).to(s["q"].dtype)


def _pairs(c):
    """Visible (query, key) pairs of one head and keys that some query sees, over the batch (lengths at their mean)."""
    n, m = c["tokens"], c["keys"]
    lo = min(m, n + m // 4) if c["ragged"] else m
    length = (lo + m) // 2
    start = 0 if n == m else length - n
    pairs, keys = 0, 0
    step = max(1, n // 512)
    for i in range(0, n, step):
        p = start + i
        hi = length if c["right"] < 0 else min(length, p + c["right"] + 1)
        first = 0 if c["left"] < 0 else min(max(0, p - c["left"]), hi)
        pairs += min(step, n - i) * (hi - first + min(c["sinks"], first))
        keys = max(keys, hi if n > 1 else hi - first + min(c["sinks"], first))
    return c["batch"] * pairs, c["batch"] * keys


def work(case):
    c = case
    size = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "rope":
        values = c["batch"] * c["tokens"] * c["heads"] * c["dim"]
        return {"bytes": 2 * values * size + 4 * c["tokens"] * c["rotary"], "flops": 3 * values}
    if c["op"] == "append":
        values = c["batch"] * c["tokens"] * (c["heads"] + 2 * c["kv_heads"]) * c["dim"]
        share = 0.5 if c["ragged"] else 1.0
        return {"bytes": share * (2 * values * size + 4 * c["batch"] * c["tokens"] * c["rotary"]), "flops": 3 * share * values}
    if c["op"] == "attend":
        pairs, keys = _pairs(c)
        rows = 2 * c["batch"] * c["tokens"] * c["heads"] * c["dim"] * size
        return {"bytes": rows + 2 * keys * c["kv_heads"] * c["dim"] * size, "flops": 4 * pairs * c["heads"] * c["dim"]}
    n, k = c["outer"], c["inner"]
    weights = n * k // 2 + n * (k // c["group"]) * (3 if c["zeros"] else 2)
    return {"bytes": weights + 4 * n + c["rows"] * (n + k) * size, "flops": 2 * c["rows"] * n * k}


def exact(case, seed):
    """The operators' definitions in 64 bits."""
    c, s = case, prepare(case, seed)
    if c["op"] == "rope":
        z = s["x"].double()
        return _turned(z, s["cos"].double()[s["positions"]], s["sin"].double()[s["positions"]] * (-1 if c["inverse"] else 1),
                       c["layout"])  # fmt: skip
    if c["op"] == "append":
        q, k, v = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), s["k_cache"].double(), s["v_cache"].double()
        starts = s["starts"].tolist()
        counts = [c["tokens"]] * c["batch"] if s["counts"] is None else s["counts"].tolist()
        for b, (first, count) in enumerate(zip(starts, counts)):
            cos, sin = s["cos"][first : first + count].double(), s["sin"][first : first + count].double()
            q[b, :, :count] = _turned(s["q"][b, :, :count].double(), cos, sin, c["layout"])
            turned = _turned(s["k"][b, :, :count].double(), cos, sin, c["layout"])
            held = {}  # the last token of each slot
            for t in range(count):
                p = first + t
                rolls = c["sinks"] >= 0 and p >= c["capacity"]
                held[c["sinks"] + (p - c["sinks"]) % (c["capacity"] - c["sinks"]) if rolls else p] = t
            if held:
                slots = torch.tensor(list(held), device="cuda")
                tokens = torch.tensor(list(held.values()), device="cuda")
                k[b][:, slots] = turned[:, tokens]
                v[b][:, slots] = s["v"][b][:, tokens].double()
        return q, k, v
    if c["op"] == "attend":
        n, d, each = c["tokens"], c["dim"], c["heads"] // c["kv_heads"]
        out = torch.zeros(c["batch"], n, c["heads"], d, dtype=torch.float64, device="cuda")
        for b, (first, length) in enumerate(zip(s["starts"].tolist(), s["lengths"].tolist())):
            for i in range(0, n, 1024):
                p = torch.arange(first + i, first + min(i + 1024, n), device="cuda")[:, None]
                lo = 0 if c["left"] < 0 else max(0, first + i - c["left"])
                hi = length if c["right"] < 0 else max(0, min(length, first + min(i + 1024, n) + c["right"]))
                early = torch.arange(0, min(lo, c["sinks"], hi), device="cuda")
                j = torch.cat([early, torch.arange(min(lo, hi), hi, device="cuda")])
                seen = torch.ones(p.shape[0], j.numel(), dtype=torch.bool, device="cuda")
                if c["right"] >= 0:
                    seen &= j <= p + c["right"]
                if c["left"] >= 0:
                    seen &= (j >= p - c["left"]) | (j < c["sinks"])
                some = seen.any(dim=1)[:, None]
                for h in range(c["heads"]):
                    k, v = s["k"][b, h // each, j].double(), s["v"][b, h // each, j].double()
                    z = (s["q"][b, h, i : i + 1024].double() @ k.T / math.sqrt(d)).masked_fill(~seen, -math.inf)
                    w = torch.softmax(torch.where(some, z, 0.0), dim=1) * some
                    out[b, i : i + 1024, h] = w @ v
        return out.flatten(2)
    x = s["x"].double()
    x = x * torch.sigmoid(x) if c["silu"] else x
    w = torch.empty(c["outer"], c["inner"], dtype=torch.float64, device="cuda")
    w[:, 0::2], w[:, 1::2] = s["packed"].remainder(16), s["packed"].div(16, rounding_mode="floor")
    w -= 8.0 if s["zero"] is None else s["zero"].double().repeat_interleave(c["group"], dim=1)
    w *= s["scale"].double().repeat_interleave(c["group"], dim=1)
    return x @ w.T + s["bias"].double()


def _turned(x, cos, sin, layout):
    """Each pair as a complex number, times e^(i angle)."""
    r = cos.shape[-1]
    out = x.clone()
    first, second = (slice(0, r), slice(r, 2 * r)) if layout == "half" else (slice(0, 2 * r, 2), slice(1, 2 * r, 2))
    z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * torch.complex(cos, sin)
    out[..., first], out[..., second] = z.real, z.imag
    return out
