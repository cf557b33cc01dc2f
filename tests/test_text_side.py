"""The text-side operators without a GPU: refusals (all before any launch), the
scaled rotary tables and the 4-bit packing."""

import ctypes
import math
import re
import struct

import pytest
import torch

from conftest import REPO
from text_side import unpacked
from test_library import _einval, lib  # noqa: F401 (lib: the built library)


@pytest.fixture(scope="module")
def K(lib):  # noqa: F811
    from iris_b200 import kernels

    return kernels


# the problem structs of include/iris_b200.h: 8-byte members, pointers as addresses
ROPE, APPEND, WINDOW, Q4 = (struct.Struct(f) for f in ("@22q", "@40q", "@29qd", "@15q"))


def test_problem_structs_are_as_packed_here():
    text = re.sub(r"/\*.*?\*/", "", (REPO / "include" / "iris_b200.h").read_text(), flags=re.S)
    for name, packing in [("rope", ROPE), ("append", APPEND), ("window", WINDOW), ("q4", Q4)]:
        body = re.search(rf"typedef struct iris_{name}_problem {{(.*?)}}", text, flags=re.S).group(1)
        fields = 0
        for line in filter(str.strip, body.split(";")):
            kind = re.match(r"\s*(const )?(iris_head_rows|void\*|float\*|int\*|int64_t|double)", line).group(2)
            fields += (4 if kind == "iris_head_rows" else 1) * (line.count(",") + 1)
        assert packing.size == 8 * fields, name


def test_c_entries_refuse_bad_arguments(lib):  # noqa: F811
    def rows(data=16, b=0, h=0, n=0):
        return data, b, h, n

    def rope(dtype=1, batch=1, heads=2, n=3, dim=64, rotary=64, table=9, layout=0, x=16):
        return "iris_rope", ROPE.pack(*rows(x), *rows(), 16, 16, 0, 0, 0, dtype, batch, heads, n, dim, rotary,
                                                   table, layout, 0), None  # fmt: skip

    for bad, message in [(dict(dtype=3), "dtype"), (dict(dim=63), "even"), (dict(rotary=66), "rotated columns"),
                         (dict(rotary=0), "rotated columns"), (dict(table=0), "table"), (dict(layout=2), "layout"),
                         (dict(x=0), "null"), (dict(n=1 << 31), "row counts"), (dict(heads=0), "row counts")]:  # fmt: skip
        assert message in _einval(lib, *rope(**bad)), bad

    def append(kv=1, capacity=8, sinks=-1, starts=16):
        return "iris_rope_append", APPEND.pack(*rows() * 6, 16, 16, starts, 0, 1, 1, 2, kv, 3, 64, 64, 9, capacity, sinks, 0, 0), None  # fmt: skip

    for bad, message in [(dict(kv=0), "head counts"), (dict(capacity=0), "slots"), (dict(sinks=8), "slots"),
                         (dict(sinks=-2), "slots"), (dict(starts=0), "null")]:  # fmt: skip
        assert message in _einval(lib, *append(**bad)), bad

    def attend(q=16, dtype=1, batch=1, heads=4, kv=2, n=3, m=5, dim=128, qn=128, kn=128, left=-1, right=0, sinks=0, scale=0.1):
        return "iris_window_attn_fwd", WINDOW.pack(
            *rows(q, n=qn), *rows(n=kn), *rows(n=128), 16, 0, 0, 0, 0, 0, 0, dtype, batch, heads, kv, n, m, dim, left, right,
            sinks, scale), None  # fmt: skip

    for bad, message in [(dict(dtype=0), "bf16 or f16"), (dict(heads=3), "multiple of heads_kv"), (dict(dim=80), "head_dim"),
                         (dict(qn=12), "16 bytes"), (dict(q=8), "16 bytes"), (dict(left=-2), "bounds"), (dict(right=-2), "bounds"),
                         (dict(sinks=-1), "bounds"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
                         (dict(scale=math.nan), "scale"), (dict(scale=math.inf), "scale"), (dict(m=1 << 30), "sizes"),
                         (dict(batch=65536), "sizes"), (dict(qn=0), "repeat"), (dict(kn=0), "repeat"), (dict(q=0), "null")]:  # fmt: skip
        assert message in _einval(lib, *attend(**bad)), bad

    def q4(x=16, dtype=1, m=1, k=128, ldx=128, group=32, n=4, out=16, out_dtype=1):
        return "iris_gemv_q4", Q4.pack(x, 16, 16, 0, 0, out, m, k, n, ldx, group, dtype, out_dtype, 0, 0), None

    for bad, message in [(dict(group=16), "groups"), (dict(m=0), "1 to 64"), (dict(m=65), "1 to 64"), (dict(k=96, group=64), "multiple"),
                         (dict(ldx=120), "size"), (dict(n=0), "1 to 64"), (dict(x=8), "aligned"), (dict(ldx=132), "aligned"),
                         (dict(dtype=3), "dtype"), (dict(out_dtype=-1), "dtype"), (dict(out=0), "null")]:  # fmt: skip
        assert message in _einval(lib, *q4(**bad)), bad
    for name in ("iris_rope", "iris_rope_append", "iris_window_attn_fwd", "iris_gemv_q4"):
        assert "null" in _einval(lib, name, None, None)


def test_workspace_is_for_split_keys_alone(lib):  # noqa: F811
    def need(batch=1, heads=4, kv=1, n=1, m=40000, dim=128, left=-1, right=0, sinks=0):
        out = ctypes.c_int64(-1)
        problem = WINDOW.pack(*[0] * 19, 1, batch, heads, kv, n, m, dim, left, right, sinks, 1.0)
        assert lib.iris_window_attn_workspace(problem, ctypes.byref(out)) == 0
        return out.value

    parts = need() // (16 * (128 + 2) * 4)  # 16 rows of sums, a maximum and a total each
    assert need() == parts * 16 * (128 + 2) * 4 and 8 < parts <= 40000 // 64
    assert need(n=4) == need() and need(dim=64) * (128 + 2) == need() * (64 + 2)
    # whole tiles, no keys or rows, one chunk, a cluster's chunks: none
    for none in (dict(n=40000), dict(m=0), dict(n=0), dict(batch=0), dict(m=64), dict(m=1028), dict(left=50), dict(batch=64, kv=4)):
        assert need(**none) == 0, none


def test_wrappers_refuse_before_any_launch(K):
    x = torch.zeros(2, 4, 3, 64)
    cos = sin = torch.zeros(9, 32)
    with pytest.raises(ValueError, match="CUDA"):
        K.rope(x, cos, sin)
    for args, kw, message in [
        ((x[0], cos, sin), {}, "head rows"),
        ((x, cos.half(), sin), {}, "FP32"),
        ((x, torch.zeros(9, 33), torch.zeros(9, 33)), {}, "tables"),
        ((x, cos, torch.zeros(9, 31)), {}, "tables"),
        ((x, torch.zeros(2, 32), torch.zeros(2, 32)), {}, "cover"),
        ((x, cos, sin, torch.zeros(4, dtype=torch.int64)), {}, "positions"),
        ((x, cos, sin, torch.zeros(3)), {}, "positions"),
        ((x, cos, sin, torch.zeros(6, dtype=torch.int32)[::2]), {}, "positions must be contiguous"),
        ((x.double(), cos, sin), {}, "dtype"),
        ((torch.zeros(2, 4, 3, 128)[..., ::2], cos, sin), {}, "contiguous"),
        ((x, cos, sin), {"layout": "both"}, "layout"),
    ]:
        with pytest.raises(ValueError, match=message):
            K.rope(*args, **kw)
    q, k, cache = torch.zeros(2, 4, 3, 64), torch.zeros(2, 2, 3, 64), torch.zeros(2, 2, 8, 64)
    starts = torch.zeros(2, dtype=torch.int32)
    good = dict(q=q, k=k, v=k, cos=cos, sin=sin, starts=starts, k_cache=cache, v_cache=cache.clone())
    with pytest.raises(ValueError, match="CUDA"):
        K.rope_append(**good)
    for bad, message in [
        (dict(k=k.half()), "one type"), (dict(v=k[:, :1]), "v must be"), (dict(starts=starts.long()), "starts"),
        (dict(starts=starts[:1]), "starts"), (dict(counts=starts.long()), "counts"), (dict(sinks=8), "rolling"),
        (dict(sinks=-1), "rolling"), (dict(k_cache=cache[:1].expand(2, 2, 8, 64)), "expanded"),
        (dict(v_cache=cache[:, :, :7]), "v_cache must be"), (dict(out=q.half()), "CUDA"),
    ]:  # fmt: skip
        with pytest.raises(ValueError, match=message):
            K.rope_append(**{**good, **bad})
    q, k = q.bfloat16(), k.bfloat16()
    with pytest.raises(ValueError, match="CUDA"):
        K.window_attention(q, k, k)
    for args, kw, message in [
        ((q.float(), k.float(), k.float()), {}, "bf16, f16"),
        ((q, k, k.half()), {}, "bf16, f16"),
        ((q[..., :48], k[..., :48], k[..., :48]), {}, "head_dim"),
        ((q, k, k[:, :, :2]), {}, "v must be"),
        ((q, k, k), {"left": -1}, "negative"),
        ((q, k, k), {"right": -3}, "negative"),
        ((q, k, k), {"sinks": -1}, "negative"),
        ((q, k, k), {"lengths": torch.zeros(3, dtype=torch.int32)}, "lengths"),
        ((q, k, k), {"starts": torch.zeros(2)}, "starts"),
    ]:
        with pytest.raises(ValueError, match=message):
            K.window_attention(*args, **kw)
    packed, scale, zero = K.pack_q4(torch.randn(6, 128), 32, symmetric=False)
    x = torch.zeros(2, 128)
    with pytest.raises(ValueError, match="CUDA"):
        K.gemv_q4(x, packed, scale, zero)
    for args, message in [
        ((x[:, :64], packed, scale, zero), "packed"), ((x, packed.int(), scale, zero), "packed"),
        ((x, packed, scale.float(), zero), "scale"), ((x, packed, scale[:5], None), "scale"),
        ((x, packed, scale, zero[:, :2]), "zero"), ((x, packed, scale, zero, torch.zeros(5)), "bias"),
        ((x, packed, scale, zero, torch.zeros(6).half()), "FP32"), ((x.t(), packed, scale, zero), "packed"),
    ]:  # fmt: skip
        with pytest.raises(ValueError, match=message):
            K.gemv_q4(*args)
    for w, group in [(torch.zeros(4, 100), 32), (torch.zeros(4, 128), 16), (torch.zeros(128), 32)]:
        with pytest.raises(ValueError, match="pack_q4"):
            K.pack_q4(w, group)


def test_wrappers_refuse_what_is_no_tensor_or_number(K):
    x, cos = torch.zeros(2, 4, 3, 64), torch.zeros(9, 32)
    for call in (lambda: K.rope(None, cos, cos), lambda: K.rope(x, [1.0], cos), lambda: K.rope(x, cos, cos, 3),
                 lambda: K.rope(x, cos, cos, out=x.numpy()), lambda: K.rope(x, cos, cos, layout=1),
                 lambda: K.rope_append(x, x, x, cos, cos, None, x, x), lambda: K.gemv_q4(x, None, x),
                 lambda: K.gemv_q4(x[0, 0], x[0, 0].byte(), x[0, 0].bfloat16(), out_dtype="f32")):  # fmt: skip
        with pytest.raises(ValueError):
            call()
    q = x.bfloat16()
    for bad in (dict(left="1"), dict(sinks=1.5), dict(scale="a"), dict(right=2**70)):
        with pytest.raises((TypeError, OverflowError)):
            K.window_attention(q, q, q, **bad)


def test_missing_module_fails_loudly(lib, monkeypatch, tmp_path):  # noqa: F811
    from iris_b200 import _lib

    monkeypatch.setattr(_lib, "_text_side", None)
    monkeypatch.setattr(_lib, "TEXT_SIDE", tmp_path / "_text_side.so")
    with pytest.raises(RuntimeError, match="not built"):
        _lib.text_side()


def test_rope_table_matches_its_formulas():
    from iris_b200.tables import rope_table

    r, length, theta = 64, 5000, 10000.0
    p = torch.arange(length, dtype=torch.float64)[:, None]
    plain = theta ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)

    def same(got, angles, magnitude=1.0):
        # one rounding to fp32 of a value of at most `magnitude`, and 64-bit angles of up to 5000 (2^-40 at most)
        for table, exact in zip(got, (angles.cos(), angles.sin())):
            assert table.dtype == torch.float32 and table.is_contiguous() and table.shape == (length, r // 2)
            assert torch.all((table.double() - magnitude * exact).abs() <= magnitude * (2.0**-24 + 2.0**-38))

    same(rope_table(r, length, theta), p * plain)
    same(rope_table(r, length, theta, scaling="linear", factor=8.0), p * plain / 8)
    ntk = rope_table(r, length, theta, scaling="ntk", factor=8.0)
    same(ntk, p * (theta * 8.0 ** (r / (r - 2))) ** (-torch.arange(0, r, 2, dtype=torch.float64) / r))
    stretched = (theta * 8.0 ** (r / (r - 2))) ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)
    assert stretched[0] == plain[0] and math.isclose(stretched[-1], plain[-1] / 8, rel_tol=1e-12)
    got = rope_table(r, length, theta, scaling="ramp", factor=4.0, trained_length=1024)
    magnitude = 0.1 * math.log(4.0) + 1
    turns = 1024 * plain / (2 * math.pi)
    # the pairs beyond either end of the ramp: kept, or divided
    kept, divided = turns > 33 * 1.4, turns < 1 / 1.4
    assert kept.any() and divided.any()
    for where, freqs in ((kept, plain), (divided, plain / 4)):
        angles = p * freqs
        for table, exact in zip(got, (angles.cos(), angles.sin())):
            assert torch.all((table.double() - magnitude * exact)[:, where].abs() <= magnitude * (2.0**-24 + 2.0**-38))
    # between the ends the angle of position 1 falls from one to the other, pair by pair
    first = (torch.atan2(got[1], got[0])[1]).double() / plain
    assert torch.all(first[1:] <= first[:-1] + 2e-6) and torch.all((first > 0.25 - 1e-6) & (first < 1 + 1e-6))
    for bad in (dict(rotary=63), dict(rotary=0), dict(length=0), dict(theta=1.0), dict(factor=0.5, scaling="linear"),
                dict(factor=2.0), dict(scaling="other"), dict(scaling="ramp", factor=2.0), dict(rotary=2, scaling="ntk")):  # fmt: skip
        with pytest.raises(ValueError):
            rope_table(**{"rotary": r, "length": length, **bad})


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("symmetric", [True, False])
def test_pack_q4_takes_the_nearest_level(K, group, symmetric):
    gen = torch.Generator().manual_seed(group)
    w = torch.randn(5, 3 * group, generator=gen)
    w[1, :group] = 0  # an empty group
    w[2] = w[2].abs() + 0.5  # one sign
    w[3, 0] = 40.0  # an outlier
    packed, scale, zero = K.pack_q4(w, group, symmetric)
    assert packed.dtype == torch.uint8 and packed.shape == (5, 3 * group // 2) and scale.dtype == torch.bfloat16
    assert (zero is None) == symmetric
    back = unpacked(packed, scale, zero).float()
    step = scale.float().repeat_interleave(group, dim=1)
    # half a level; at the range's ends the bf16 scale may fall short by 2^-8 of up to 15 levels, and a whole zero point
    # is up to half a level off
    assert torch.all((back - w).abs() <= step * (0.5 + 15 * 2.0**-8 + (0 if symmetric else 0.5)) + 1e-6)
    assert torch.all(back[1, :group] == 0)


def test_kernels_that_start_early_use_coherent_loads():
    """A kernel launched with launch_early lives while its predecessor writes what it will read: a non-coherent load
    (data that nobody writes as long as the kernel lives) may be served from before the wait."""
    early = [f for f in sorted((REPO / "iris-3b-metal_b200" / "csrc").glob("*.cu")) if "launch_early(" in f.read_text()]
    assert {"q4.cu", "rope.cu", "window.cu"} <= {f.name for f in early}
    for f in early:
        code = re.sub(r"//.*", "", f.read_text())
        assert not re.search(r"__ldg|__ldcs|ld\.global\.nc|__restrict__", code), f.name


def test_prompt_tiles_wait_for_their_copies_whoever_gives_up():
    """The thread that issued a tile's last copies waits for them on every path: another warp may give up (and the CTA
    end) after this one has issued everything."""
    code = (REPO / "iris-3b-metal_b200" / "csrc" / "window.cu").read_text()
    issue = code[code.index("--- TMA") : code.index("--- MMA")]
    guard, drain = re.search(r"\n    if \(([^\n]*)\) \{[^\n]*\n      int dummy = 0;(.*?)\n    \}\n", issue, flags=re.S).groups()
    assert guard == "lane == 0 && iters > 0"
    assert all(f"mbar_wait(&s->{bar}" in drain for bar in ("q_full", "k_full", "v_full", "v_tail"))


def test_outputs_that_would_race_are_refused(K):
    """Two elements in one place, or an output in what other threads of the call still read (before any device check)."""
    cos = sin = torch.zeros(9, 32)
    buf = torch.zeros(4096)
    x = buf[:1536].view(2, 4, 3, 64)

    def refused(message, call, *args, **kw):
        with pytest.raises(ValueError, match=message):
            call(*args, **kw)

    refused("CUDA", K.rope, x, cos, sin, out=x)  # in place is allowed: it gets as far as the device
    refused("CUDA", K.rope, x, cos, sin, out=x.view(2, 4, 3, 64))
    refused("CUDA", K.rope, x, cos, sin, out=buf[2048:3584].view(2, 4, 3, 64))
    refused("x itself", K.rope, x, cos, sin, out=buf[64:1600].view(2, 4, 3, 64))
    refused("x itself", K.rope, x, cos, sin, out=buf[:1536].view(2, 3, 4, 64).transpose(1, 2))
    refused("CUDA", K.rope, buf[:0].view(2, 4, 0, 64), cos, sin, out=buf[:0].view(2, 4, 0, 64))
    for strides in [(768, 192, 32, 1), (192, 192, 64, 1), (768, 64, 64, 1)]:  # rows that overlap without a stride of 0
        refused("overlap|CUDA", K.rope, x, cos, sin, out=torch.zeros(4096).as_strided((2, 4, 3, 64), strides))
    packed = torch.zeros(2, 3, 12, 64).transpose(1, 2)  # interleaved heads of one buffer are apart
    refused("CUDA", K.rope, packed[:, :4], cos, sin, out=packed[:, 4:8])

    q, k, v = torch.zeros(2, 4, 3, 64), torch.zeros(2, 2, 3, 64), torch.zeros(2, 2, 3, 64)
    caches = torch.zeros(2, 2, 2, 8, 64)
    good = dict(q=q, k=k, v=v, cos=cos, sin=sin, starts=torch.zeros(2, dtype=torch.int32), k_cache=caches[0], v_cache=caches[1])
    refused("CUDA", K.rope_append, **good)
    refused("CUDA", K.rope_append, **{**good, "out": q})
    refused("CUDA", K.rope_append, **{**good, "v": k})
    for bad in (dict(v_cache=caches[0]), dict(k=caches[0, :, :, :3]), dict(v=caches[1, :, :, :3]), dict(out=caches.view(-1)[:1536].view_as(q)),
                dict(out=q.view(2, 3, 4, 64).transpose(1, 2)), dict(k_cache=caches.view(-1)[64:2112].view(2, 2, 8, 64)),
                dict(k=q.view(-1)[:768].view_as(k), out=q)):  # fmt: skip
        refused("share", K.rope_append, **{**good, **bad})

    rows = torch.zeros(2, 3, 256, dtype=torch.bfloat16)
    q, k = rows.view(2, 3, 4, 64).transpose(1, 2), torch.zeros(2, 2, 3, 64, dtype=torch.bfloat16)
    refused("CUDA", K.window_attention, q, k, k, out=rows)  # q's own rows
    refused("own rows", K.window_attention, rows.view(2, 4, 3, 64), k, k, out=rows)
    refused("CUDA", K.window_attention, rows[:, :1].view(2, 4, 1, 64), k, k, out=rows[:, :1])
    refused("k or v", K.window_attention, q[:, :2], k, rows.view(2, 2, 6, 64)[:, :, :3], out=rows[..., :128])
    refused("k or v", K.window_attention, q[:, :2], q, q, out=rows[..., :128])
    refused("overlap|CUDA", K.window_attention, q, k, k, out=torch.zeros(2048, dtype=torch.bfloat16).as_strided((2, 3, 256), (768, 64, 1)))


@pytest.mark.parametrize("rotary, theta, trained, fast, slow", [
    (128, 1e4, 131072, 32.0, 1.0),  # the slowest pair still turns 2.4 times
    (128, 1e4, 4096, 32.0, 1.0),
    (64, 1e4, 1 << 22, 32.0, 1.0),  # even the slowest pair turns more than 32 times
    (64, 1e6, 8192, 16.0, 2.0),
    (32, 1e4, 100, 32.0, 1.0),  # the fastest pair turns 16 times
    (32, 1e4, 5, 32.0, 1.0),  # no pair turns once
])  # fmt: skip
def test_rope_table_ramp_at_every_trained_length(rotary, theta, trained, fast, slow):
    """Pair by pair: kept from `fast` turns on, divided up to `slow`, in between by the pair's index."""
    from iris_b200.tables import rope_table

    factor, positions = 4.0, 40
    cos, sin = rope_table(rotary, positions, theta, scaling="ramp", factor=factor, trained_length=trained, fast_turns=fast, slow_turns=slow)
    magnitude = 0.1 * math.log(factor) + 1

    def index(turns):  # trained theta^(-2 i / rotary) = 2 pi turns
        return rotary / 2 * math.log(trained / (2 * math.pi * turns), theta)

    first, last = max(0, math.floor(index(fast))), math.ceil(index(slow))
    shares = []
    for i in range(rotary // 2):
        freq = theta ** (-2 * i / rotary)
        turns = trained * freq / (2 * math.pi)
        share = 0.0 if turns >= fast else 1.0 if turns <= slow else (i - first) / (last - first)
        share = min(1.0, max(0.0, share))
        freq = freq * (1 - share) + freq / factor * share
        for p in (1, positions - 1):
            # one rounding to fp32 of a value of at most 1.2, and a 64-bit angle of at most 40
            assert abs(float(cos[p, i]) - magnitude * math.cos(p * freq)) <= 2.0**-23
            assert abs(float(sin[p, i]) - magnitude * math.sin(p * freq)) <= 2.0**-23
        shares.append(share)
    assert shares == sorted(shares)
    assert (max(shares) < 1) == (index(slow) > rotary / 2 - 1) and (min(shares) == 1) == (index(slow) <= 0)


@pytest.mark.parametrize("symmetric", [True, False])
def test_pack_q4_of_a_parameter_keeps_no_graph(K, symmetric):
    """Packed weights stand alone: nothing of them holds the parameter's values or its autograd graph."""
    w = torch.nn.Linear(64, 6).weight
    packed = K.pack_q4(w, 32, symmetric)
    for got, plain in zip(packed, K.pack_q4(w.detach(), 32, symmetric)):
        if got is not None:
            assert not got.requires_grad and got.grad_fn is None and torch.equal(got, plain)


def test_scale_beyond_the_range_is_refused(lib):  # noqa: F811
    """Scores are taken times scale log2(e): past fp32 a score of 0 would be NaN."""
    def attend(scale):
        heads = (16, 0, 0, 128)
        return WINDOW.pack(*heads * 3, 16, 0, 0, 0, 0, 0, 0, 1, 1, 4, 2, 0, 5, 128, -1, 0, 0, scale), None  # no rows: nothing runs

    for scale in (2.4e38, 3.4e38, 1e39, 1e-50):
        assert "scale" in _einval(lib, "iris_window_attn_fwd", *attend(scale)), scale
    for scale in (2.3e38, 1e-37):
        assert lib.iris_window_attn_fwd(*attend(scale)) == 0


def test_the_module_is_for_one_python_and_torch(lib, monkeypatch):  # noqa: F811
    """Compiled against torch's and CPython's own types: another version does not load it, and builds its own."""
    from iris_b200 import _lib, build

    assert build.MODULE == _lib.TEXT_SIDE == _lib.text_side_path() and _lib.TEXT_SIDE.exists()
    for target, name, value in [(torch, "__version__", "9.9.0"), (_lib.sysconfig, "get_config_var", lambda name: "cpython-399")]:
        with monkeypatch.context() as m:
            m.setattr(target, name, value)
            other = _lib.text_side_path()
            assert other != _lib.TEXT_SIDE and not other.exists()
            m.setattr(build, "MODULE", other)
            assert not build.module_up_to_date()
            m.setattr(_lib, "TEXT_SIDE", other)
            m.setattr(_lib, "_text_side", None)
            with pytest.raises(RuntimeError, match="not built"):
                _lib.text_side()


def test_strides_of_lone_entries_are_not_looked_at(lib):  # noqa: F811
    """Up to the check that refuses a missing output, which comes after those of the strides."""
    for stride in (12, -128, 1 << 45):
        for q, k, n, m in [((16, 0, 0, stride), (16, 0, 0, 128), 1, 5), ((16, stride, 0, 128), (16, stride, 0, 128), 3, 5),
                           ((16, 0, 0, 128), (16, 0, stride, stride), 3, 1)]:  # fmt: skip
            problem = WINDOW.pack(*q, *k, *k, 0, 0, 0, 0, 0, 0, 0, 1, 1, 4, 1, n, m, 128, -1, 0, 0, 0.1)
            assert "null" in _einval(lib, "iris_window_attn_fwd", problem, None), (q, k)
