"""The text-side operators on the B200 against their definitions in 64 bits, each
element within what its roundings allow (text_side.py)."""

import math

import pytest
import torch

from conftest import requires_gpu
from text_side import assert_attends, assert_q4, assert_turned, attention, turned, visible

pytestmark = requires_gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
ERR_BAD_ARGUMENT = 2


@pytest.fixture(scope="module")
def K():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from iris_b200 import kernels

    return kernels


def normal(seed, *shape, dtype=F32):
    return torch.randn(*shape, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)).to(dtype)


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def table(rotary, length, **kw):
    from iris_b200.tables import rope_table

    return rope_table(rotary, length, device="cuda", **kw)


def packed_heads(seed, b, n, h, kv, d, dtype):
    """q, k, v views of one projection's rows."""
    rows = normal(seed, b, n, (h + 2 * kv) * d, dtype=dtype).view(b, n, h + 2 * kv, d).transpose(1, 2)
    return rows[:, :h], rows[:, h : h + kv], rows[:, h + kv :]


# ------------------------------------------------------------------- rope
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim, rotary", [(128, 128), (64, 64), (128, 32), (80, 40), (96, 24), (6, 6), (10, 2), (2, 2)])
def test_rope(K, dtype, layout, dim, rotary):
    b, h, n = 3, 5, 7
    cos, sin = table(rotary, 50)
    x = packed_heads(dim + rotary, b, n, h, 1, dim, dtype)[0]
    before = x.clone()
    order = torch.randperm(43, device="cuda")
    for positions in (None, order[:n], (order[: b * n].view(b, n) + 5).int(), order[:n].expand(b, n)):
        at = torch.arange(n, device="cuda") if positions is None else positions.long()
        c, s = cos[at], sin[at]
        if at.dim() == 2:
            c, s = c[:, None], s[:, None]
        got = K.rope(x, cos, sin, positions, layout=layout)
        assert got.is_contiguous() and torch.equal(x, before)
        assert_turned(got, x, c, s, layout)
        back = K.rope(x, cos, sin, positions, layout=layout, inverse=True)
        assert_turned(back, x, c, -s, layout)
    # onto its own rows, and into rows of another order
    own = x.clone()
    assert K.rope(own, cos, sin, layout=layout, out=own) is own
    other = torch.empty(b, n, h, dim, device="cuda", dtype=dtype).transpose(1, 2)
    K.rope(x, cos, sin, layout=layout, out=other)
    assert torch.equal(own, other) and torch.equal(own, K.rope(x, cos, sin, layout=layout))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shift", [1, 2, 4])
def test_rope_reads_rows_at_any_alignment(K, dtype, shift):
    cos, sin = table(64, 9)
    flat = normal(shift, 2 * 3 * 9 * 72 + 8, dtype=dtype)
    x = flat[shift : shift + 2 * 3 * 9 * 72].view(2, 3, 9, 72)[..., :64]
    aligned = x.contiguous()
    assert torch.equal(K.rope(x, cos, sin), K.rope(aligned, cos, sin))
    out = torch.zeros(2, 3, 9, 64 + shift, device="cuda", dtype=dtype)
    K.rope(x, cos, sin, out=out[..., shift:])
    assert torch.equal(out[..., shift:], K.rope(aligned, cos, sin)) and torch.all(out[..., :shift] == 0)


@pytest.mark.parametrize("shift", [1, 2])
def test_rope_reads_tables_at_any_alignment(K, shift):
    cos, sin = table(64, 9)
    x = normal(1, 2, 3, 9, 64, dtype=BF16)
    moved = [torch.cat([torch.zeros(shift, device="cuda"), t.flatten()])[shift:].view(9, 32) for t in (cos, sin)]
    assert all(t.data_ptr() % 16 for t in moved)
    for layout in ("half", "interleaved"):
        assert torch.equal(K.rope(x, *moved, layout=layout), K.rope(x, cos, sin, layout=layout))


def test_rope_sizes(K):
    cos, sin = table(64, 70000)
    for b, h, n in [(1, 1, 1), (1, 300, 1), (2, 1, 70000), (0, 3, 4), (2, 3, 0), (600, 2, 3)]:
        x = normal(n, b, h, n, 64, dtype=BF16)
        got = K.rope(x, cos, sin, layout="half")
        assert got.shape == x.shape
        assert_turned(got, x, cos[:n], sin[:n], "half")


def test_rope_far_positions_and_their_gradient(K):
    """The rotation is orthogonal: <R x, y> = <x, R^-1 y>, so `inverse` is the gradient's map."""
    cos, sin = table(128, 200001, theta=1000000.0)
    x, y = normal(1, 1, 4, 33, 128), normal(2, 1, 4, 33, 128)
    at = 200000 - 37 * torch.arange(33, device="cuda")
    turned_x, back = K.rope(x, cos, sin, at, layout="half"), K.rope(y, cos, sin, at, layout="half", inverse=True)
    a, b = (turned_x.double() * y.double()).sum(), (x.double() * back.double()).sum()
    # each product's factor is off by 2^-22 of its size at most
    assert abs(a - b) <= 2.0**-21 * (x.abs().double() * y.abs().double()).sum() * 2
    step = K.rope(x + y, cos, sin, at, layout="half").double() - turned_x.double()  # linear: a difference is the image
    assert_close = (step - K.rope(y, cos, sin, at, layout="half").double()).abs()
    assert torch.all(assert_close <= 2.0**-20 * (x.abs().amax() + y.abs().amax()))


def test_rope_positions_outside_the_tables(K):
    cos, sin = table(64, 8)
    x = normal(3, 1, 2, 4, 64, dtype=BF16)
    K.device_error()
    got = K.rope(x, cos, sin, torch.tensor([3, -1, 7, 8], device="cuda"))
    assert K.device_error() & ERR_BAD_ARGUMENT and not K.device_error()
    assert torch.isnan(got[:, :, 1]).all() and torch.isnan(got[:, :, 3]).all()
    at = torch.tensor([3, 7], device="cuda")
    assert_turned(got[:, :, [0, 2]], x[:, :, [0, 2]], cos[at], sin[at], "interleaved")


# ----------------------------------------------------------------- append
def appended(k_cache, v_cache, k, v, cos, sin, starts, counts, sinks, layout):
    """The caches afterwards, row by row: fp64 keys (None where untouched) and values."""
    capacity = k_cache.shape[2]
    source = {}
    for b, (first, count) in enumerate(zip(starts, counts)):
        for t in range(count):
            p = first + t
            if sinks is None:
                slot = p
            else:
                slot = p if p < capacity else sinks + (p - sinks) % (capacity - sinks)
            if slot < capacity:
                source[b, slot] = (t, p)
    return source


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize(
    "n, capacity, sinks, starts, counts",
    [
        (1, 16, None, [15, 0, 3], None),
        (5, 16, None, [11, 0, 3], [5, 0, 2]),
        (1, 12, 4, [11, 12, 30011], None),
        (1, 12, 0, [0, 12, 23], [1, 0, 1]),
        (30, 12, 4, [0, 7, 1000], [30, 9, 25]),  # a prompt longer than the cache: its last rows and first four stay
        (9, 7, 6, [0, 2, 50], None),  # one slot turns
        (4, 33, 2, [0, 29, 5], [4, 4, 1]),
    ],
)
def test_rope_append(K, dtype, layout, n, capacity, sinks, starts, counts):
    b, h, kv, d, rotary = 3, 6, 2, 64, 32
    cos, sin = table(rotary, max(starts) + n)
    q, k, v = packed_heads(n + capacity, b, n, h, kv, d, dtype)
    k_cache, v_cache = normal(1, b, kv, capacity, d, dtype=dtype), normal(2, b, capacity, kv, d, dtype=dtype).transpose(1, 2)
    k_old, v_old = k_cache.clone(), v_cache.clone()
    K.device_error()
    kw = dict(sinks=sinks, counts=None if counts is None else int32(counts), layout=layout)
    got = K.rope_append(q, k, v, cos, sin, int32(starts), k_cache, v_cache, **kw)
    assert K.device_error() == 0
    rows = [n] * b if counts is None else counts
    source = appended(k_cache, v_cache, k, v, cos, sin, starts, rows, sinks, layout)
    for s in range(b):
        at = slice(starts[s], starts[s] + rows[s])
        assert_turned(got[s, :, : rows[s]], q[s, :, : rows[s]], cos[at], sin[at], layout)
        assert torch.all(got[s, :, rows[s] :] == 0)
        for slot in range(capacity):
            if (s, slot) not in source:
                assert torch.equal(k_cache[s, :, slot], k_old[s, :, slot])
                assert torch.equal(v_cache[s, :, slot], v_old[s, :, slot])
                continue
            t, p = source[s, slot]
            assert_turned(k_cache[s, :, slot], k[s, :, t], cos[p], sin[p], layout)
            assert torch.equal(v_cache[s, :, slot], v[s, :, t])
    # a given out keeps its rows behind the counts; onto q's own rows
    kept = normal(5, b, n, h, d, dtype=dtype).transpose(1, 2)
    before = kept.clone()
    K.rope_append(q, k, v, cos, sin, int32(starts), k_cache, v_cache, out=kept, **kw)
    for s in range(b):
        assert torch.equal(kept[s, :, : rows[s]], got[s, :, : rows[s]])
        assert torch.equal(kept[s, :, rows[s] :], before[s, :, rows[s] :])
    own = q.clone()
    K.rope_append(own, k, v, cos, sin, int32(starts), k_cache, v_cache, out=own, **kw)
    for s in range(b):
        assert torch.equal(own[s, :, : rows[s]], got[s, :, : rows[s]])


def test_rope_append_past_the_cache_and_the_tables(K):
    cos, sin = table(64, 20)
    q, k, v = packed_heads(4, 3, 2, 2, 1, 64, BF16)
    k_cache, v_cache = torch.zeros(3, 1, 8, 64, device="cuda", dtype=BF16), torch.zeros(3, 1, 8, 64, device="cuda", dtype=BF16)
    K.device_error()
    got = K.rope_append(q, k, v, cos, sin, int32([7, 19, -1]), k_cache, v_cache)
    assert K.device_error() & ERR_BAD_ARGUMENT
    assert_turned(got[0], q[0], cos[7:9], sin[7:9], "interleaved")
    assert torch.equal(v_cache[0, :, 7], v[0, :, 0]) and torch.all(v_cache[0, :, :7] == 0)  # position 8 has no slot
    assert torch.isnan(got[1, :, 1]).all() and not torch.isnan(got[1, :, 0]).any()
    assert torch.isnan(got[2, :, 0]).all() and torch.all(v_cache[1] == 0)
    assert torch.equal(v_cache[2, :, 0], v[2, :, 1]) and torch.all(v_cache[2, :, 1:] == 0)


# -------------------------------------------------------------- attention
SHAPES = [  # n, n_kv, heads, kv_heads
    (1, 1, 1, 1), (1, 40, 5, 1), (1, 257, 8, 2), (1, 1028, 20, 5), (1, 700, 16, 1), (1, 65, 40, 2), (3, 90, 12, 4), (4, 4, 2, 2),
    (17, 17, 4, 4), (100, 100, 4, 1), (128, 128, 2, 1), (129, 129, 3, 1), (300, 300, 4, 2), (257, 640, 2, 2), (5, 1000, 6, 2),
    (40, 41, 6, 6), (513, 513, 3, 3),
]  # fmt: skip
MASKS = [  # left, right, sinks
    (None, 0, 0), (None, None, 0), (0, 0, 0), (7, 0, 3), (100, 0, 4), (63, 64, 0), (20, 150, 130), (0, None, 1), (500, 0, 0),
]


@pytest.mark.parametrize("dtype, dim", [(BF16, 128), (F16, 128), (BF16, 64), (F16, 64)])
@pytest.mark.parametrize("n, n_kv, heads, kv_heads", SHAPES)
def test_window_attention(K, dtype, dim, n, n_kv, heads, kv_heads):
    b = 2
    if n == n_kv:
        q, k, v = packed_heads(n, b, n, heads, kv_heads, dim, dtype)
    else:
        q = normal(n, b, n, heads, dim, dtype=dtype).transpose(1, 2)
        k, v = normal(n + 1, b, kv_heads, n_kv, dim, dtype=dtype), normal(n + 2, b, kv_heads, n_kv, dim, dtype=dtype)
    for left, right, sinks in MASKS:
        got = K.window_attention(q, k, v, left=left, right=right, sinks=sinks)
        assert got.shape == (b, n, heads * dim) and got.is_contiguous()
        assert_attends(got, q, k, v, left=left, right=right, sinks=sinks)


@pytest.mark.parametrize("dtype, dim", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("n, n_kv", [(1, 300), (1, 1500), (6, 300), (300, 300), (140, 530)])
def test_window_attention_lengths_and_starts(K, dtype, dim, n, n_kv):
    """Empty samples, one key, a length beyond the keys, queries before and far behind them."""
    lengths = int32([0, 1, n_kv // 2, n_kv, n_kv + 50, -3, n_kv - 1])
    starts = int32([0, 0, n_kv // 2 - n, n_kv - n, n_kv, 5, -2])
    q = normal(7, 7, 6, n, dim, dtype=dtype)
    k, v = normal(8, 7, 2, n_kv, dim, dtype=dtype), normal(9, 7, 2, n_kv, dim, dtype=dtype)
    for left, right, sinks in [(None, 0, 0), (30, 0, 0), (30, 5, 4), (None, None, 0), (0, 0, 300), (3, 1, 0)]:
        got = K.window_attention(q, k, v, left=left, right=right, sinks=sinks, starts=starts, lengths=lengths)
        assert torch.all(got[0] == 0) and torch.all(got[5] == 0)
        assert_attends(got, q, k, v, left=left, right=right, sinks=sinks, starts=starts, lengths=lengths)
    # positions so far off that no key, or only the first ones, are seen
    far = int32([2**31 - 1] * 4 + [-(2**31)] * 3)
    for sinks in (0, 3):
        got = K.window_attention(q, k, v, left=9, right=0, sinks=sinks, starts=far, lengths=lengths)
        assert_attends(got, q, k, v, left=9, right=0, sinks=sinks, starts=far, lengths=lengths)
        assert torch.all(got[4:] == 0)


@pytest.mark.parametrize("dtype, dim", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("n, heads", [(1, 1), (1, 5), (1, 16), (3, 7), (17, 1)])
def test_every_number_of_chunks(K, dtype, dim, n, heads):
    """A chunk of 64 keys more each time: clusters of two to eight CTAs, few and many rows of the tile, and chunks that
    see nothing (a length inside the first one)."""
    for n_kv in range(50, 640, 64):
        q = normal(n_kv, 2, heads, n, dim, dtype=dtype)
        k, v = normal(1, 2, 1, n_kv, dim, dtype=dtype), normal(2, 2, 1, n_kv, dim, dtype=dtype)
        lengths = int32([n_kv, 30])
        got = K.window_attention(q, k, v, right=None, lengths=lengths)
        assert_attends(got, q, k, v, right=None, lengths=lengths)


@pytest.mark.parametrize("dtype, dim", [(BF16, 128), (F16, 128), (BF16, 64)])
@pytest.mark.parametrize("b, n, n_kv, heads, kv_heads", [(1, 1, 20000, 4, 1), (3, 1, 9001, 8, 8), (1, 5, 30000, 8, 2), (40, 1, 700, 8, 4),
                                                         (2, 1, 4097, 24, 1), (1, 33, 5000, 6, 2), (1, 200, 3001, 3, 3)])  # fmt: skip
def test_long_caches(K, dtype, dim, b, n, n_kv, heads, kv_heads):
    """Enough keys that they are split: over a cluster, over more parts and a join, in several waves, for several row
    tiles of a key head; samples of very different lengths."""
    q = normal(1, b, heads, n, dim, dtype=dtype)
    k, v = normal(2, b, kv_heads, n_kv, dim, dtype=dtype), normal(3, b, kv_heads, n_kv, dim, dtype=dtype)
    lengths = int32([max(1, n_kv - 977 * i) if i % 3 else n_kv for i in range(b)])
    for left, sinks in [(None, 0), (2000, 5)]:
        got = K.window_attention(q, k, v, left=left, sinks=sinks, starts=lengths - n, lengths=lengths)
        assert_attends(got, q, k, v, left=left, sinks=sinks, starts=lengths - n, lengths=lengths)
    k[:, :, -1], v[:, :, -1] = math.nan, math.nan  # the last slot is not written yet
    got = K.window_attention(q, k, v, starts=lengths - n - 1, lengths=(lengths - 1).clamp_max(n_kv - 1))
    assert torch.isfinite(got).all()


def test_kernels_are_counted(K):
    from iris_b200 import _lib

    q, k = normal(1, 1, 4, 1, 128, dtype=BF16), normal(2, 1, 1, 40000, 128, dtype=BF16)
    cos, sin = table(128, 1)

    def counted(call):
        before = _lib.launch_count()
        call()
        return _lib.launch_count() - before

    assert counted(lambda: K.window_attention(q, k[:, :, :64], k[:, :, :64])) == 1
    assert counted(lambda: K.window_attention(q, k, k)) == 2
    assert counted(lambda: K.rope(q, cos, sin)) == 1 and counted(lambda: K.rope(q[:, :, :0], cos, sin)) == 0
    w = K.pack_q4(normal(3, 64, 128), 64)
    assert counted(lambda: K.gemv_q4(q[0, :, 0], *w)) == 1


@pytest.mark.parametrize("dtype, dim", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("n, n_kv", [(1, 700), (4, 300), (300, 300), (200, 450)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_masked_places_may_hold_anything(K, dtype, dim, n, n_kv, bad):
    """NaN and infinities behind the lengths, and in keys that some queries do not see."""
    q = normal(1, 3, 4, n, dim, dtype=dtype)
    k, v = normal(2, 3, 2, n_kv, dim, dtype=dtype), normal(3, 3, 2, n_kv, dim, dtype=dtype)
    lengths, starts = int32([n_kv - 77, 5, 130]), int32([max(0, n_kv - 77 - n), 0, 100])
    for s in range(3):
        k[s, :, int(lengths[s]) :] = bad
        v[s, :, int(lengths[s]) :] = bad
    got = K.window_attention(q, k, v, left=60, sinks=3, starts=starts, lengths=lengths)
    assert torch.isfinite(got).all()
    assert_attends(got, q, k, v, left=60, sinks=3, starts=starts, lengths=lengths)
    if n > 100:  # one key in the middle of a tile: the rows that see it follow the formula, the others are untouched
        k, v = normal(2, 3, 2, n_kv, dim, dtype=dtype), normal(3, 3, 2, n_kv, dim, dtype=dtype)
        clean = K.window_attention(q, k, v, left=60, sinks=3)
        v[1, 1, n_kv - 90] = bad
        got = K.window_attention(q, k, v, left=60, sinks=3)
        full = torch.full((3,), n_kv, device="cuda")
        seen = visible(n, n_kv, full - n, full, 60, 0, 3)[1, :, n_kv - 90]
        assert seen.any() and not seen.all()
        rows = got.view(3, n, 4, dim)
        assert torch.equal(got[0], clean[0]) and torch.equal(got[2], clean[2])
        assert torch.equal(rows[1, :, :2], clean.view(3, n, 4, dim)[1, :, :2])
        if math.isnan(bad):
            assert torch.isnan(rows[1, :, 2:][seen]).all()
        else:
            assert torch.all(rows[1, :, 2:][seen] == bad)
        v[1, 1, n_kv - 90] = 0  # finite again: what the untouched rows are held to
        assert torch.isfinite(rows[1, :, 2:][~seen]).all()
        unseen = torch.where(seen[:, None, None], 0, rows[1])
        exact, allowed = attention(q[1:2], k[1:2], v[1:2], visible(n, n_kv, full - n, full, 60, 0, 3)[1:2], dim**-0.5)
        off = (unseen.double() - torch.where(seen[:, None, None], 0, exact[0])).abs()
        assert torch.all(off <= allowed[0])


@pytest.mark.parametrize("n", [1, 200])
def test_infinite_and_nan_scores(K, n):
    """As softmax has them: a NaN or +inf score makes the row NaN, a -inf one has no weight, all -inf is 0 / 0."""
    q, k, v = normal(1, 1, 2, n, 64, dtype=BF16), normal(2, 1, 1, 200, 64, dtype=BF16), normal(3, 1, 1, 200, 64, dtype=BF16)
    q = q.abs() + 0.1
    for value, expect_nan in ((math.nan, True), (math.inf, True), (-math.inf, False)):
        kk = k.clone()
        kk[:, :, 3] = value
        got = K.window_attention(q, kk, v, right=None)
        assert torch.isnan(got).all() if expect_nan else torch.isfinite(got).all()
        if not expect_nan:
            keep = torch.arange(200, device="cuda") != 3
            assert_attends(got, q, k[:, :, keep], v[:, :, keep], right=None)
    assert torch.isnan(K.window_attention(q, torch.full_like(k, -math.inf), v, right=None)).all()


@pytest.mark.parametrize("n", [1, 5, 300])
def test_large_scores(K, n):
    """Scores of several hundred, and rows that grow from key to key: the running maximum has to follow."""
    q, k, v = normal(1, 1, 2, n, 128, dtype=BF16), normal(2, 1, 1, 900, 128, dtype=BF16), normal(3, 1, 1, 900, 128, dtype=BF16)
    k = k * torch.linspace(0.1, 12, 900, device="cuda")[:, None].to(BF16)
    for scale in (0.088, 1.0, 1e-6):
        got = K.window_attention(q, k, v, right=None, scale=scale)
        assert_attends(got, q, k, v, right=None, scale=scale)


@pytest.mark.parametrize("n", [1, 300])
def test_window_attention_strides(K, n):
    """Broadcast keys, rows of other orders, lone rows with odd strides, an out with wider rows."""
    dim, dtype = 128, BF16
    q = normal(1, 2, 4, n, dim, dtype=dtype)
    k, v = normal(2, 1, 1, 300, dim, dtype=dtype), normal(3, 300, 2, dim, dtype=dtype)
    kk, vv = k.expand(2, 2, 300, dim), v.transpose(0, 1)[None].expand(2, 2, 300, dim)
    got = K.window_attention(q, kk, vv, right=None)
    assert torch.equal(got, K.window_attention(q, kk.contiguous(), vv.contiguous(), right=None))
    with pytest.raises(ValueError, match="repeat"):
        K.window_attention(q, kk, v[:1].transpose(0, 1)[None].expand(2, 2, 300, dim), right=None)
    wide = normal(4, 2, n, 4 * dim + 24, dtype=dtype)
    before = wide.clone()
    K.window_attention(q, kk, vv, right=None, out=wide[..., 8 : 8 + 4 * dim])
    assert torch.equal(wide[..., 8 : 8 + 4 * dim], K.window_attention(q, kk, vv, right=None))
    assert torch.equal(wide[..., :8], before[..., :8]) and torch.equal(wide[..., 8 + 4 * dim :], before[..., 8 + 4 * dim :])
    lone = q[:1, :2].as_strided((1, 2, 1, dim), (3, dim * n, 5, 1))
    assert torch.equal(K.window_attention(lone, k, k), K.window_attention(lone.contiguous(), k, k))
    with pytest.raises(ValueError, match="16 bytes"):
        flat = normal(5, 2 * 300 * dim + 8, dtype=dtype)
        K.window_attention(q, flat[4 : 4 + 300 * dim].view(1, 1, 300, dim).expand(2, 2, 300, dim), vv)
    with pytest.raises(ValueError, match="expanded"):
        K.window_attention(q, kk, vv, out=wide[:1, :, : 4 * dim].expand(2, n, 4 * dim))


def test_offsets_beyond_32_bits(K):
    """Keys whose element offsets pass 2^31, for the attention and the append."""
    room = torch.empty(20 * 2**27 + 1024, device="cuda", dtype=BF16)
    k = room.as_strided((1, 1, 20, 128), (0, 0, 2**27, 1))
    v = room.as_strided((1, 1, 20, 128), (0, 0, 2**27, 1), 256)
    kk, vv = normal(1, 1, 1, 20, 128, dtype=BF16), normal(2, 1, 1, 20, 128, dtype=BF16)
    k.copy_(kk)
    v.copy_(vv)
    for n in (1, 20):
        q = normal(3, 1, 4, n, 128, dtype=BF16)
        assert torch.equal(K.window_attention(q, k, v), K.window_attention(q, kk, vv))
    cos, sin = table(128, 32)
    q, new, _ = packed_heads(4, 1, 3, 2, 1, 128, BF16)
    K.rope_append(q, new, new, cos, sin, int32([17]), k, v)
    K.rope_append(q, new, new, cos, sin, int32([17]), kk, vv)
    assert torch.equal(k, kk) and torch.equal(v, vv)
    assert torch.equal(K.rope(k, cos, sin), K.rope(kk, cos, sin))


def test_no_rows(K):
    q, k = torch.zeros(2, 4, 0, 64, device="cuda", dtype=BF16), torch.zeros(2, 2, 5, 64, device="cuda", dtype=BF16)
    assert K.window_attention(q, k, k).shape == (2, 0, 256)
    q = torch.ones(2, 4, 3, 64, device="cuda", dtype=BF16)
    out = torch.full((2, 3, 256), 7.0, device="cuda", dtype=BF16)
    assert torch.all(K.window_attention(q, k[:, :, :0], k[:, :, :0], out=out) == 0)  # no keys at all


# --------------------------------------------------------------------- q4
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m", [1, 2, 3, 5, 8, 9, 16, 17, 64])
def test_gemv_q4(K, dtype, group, m):
    for n, k, symmetric, biased in [(1, group, True, False), (17, 3 * group, False, True), (130, 1280, True, True),
                                    (515, 21 * group, False, False), (64, 2560, True, True), (2561, 7 * 128, False, True)]:  # fmt: skip
        packed, scale, zero = K.pack_q4(normal(n + k, n, k), group, symmetric)
        bias = normal(9, n) if biased else None
        x = normal(m, m, k + 8, dtype=dtype)[:, :k]  # rows wider than K
        for silu_in, silu_out in [(False, False), (True, False), (False, True)]:
            got = K.gemv_q4(x, packed, scale, zero, bias, silu_in=silu_in, silu_out=silu_out)
            assert got.dtype == dtype and got.shape == (m, n)
            assert_q4(got, x, packed, scale, zero, bias, silu_in, silu_out)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m, n, k", [(1, 40, 57344), (16, 70, 20480), (64, 33, 16384), (9, 300, 30720)])
def test_gemv_q4_long_rows(K, dtype, m, n, k):
    """Rows of x that shared memory takes in several pieces."""
    packed, scale, zero = K.pack_q4(normal(n, n, k), 128, False)
    x = normal(m, m, k, dtype=dtype)
    assert_q4(K.gemv_q4(x, packed, scale, zero, out_dtype=F32), x, packed, scale, zero, None)


@pytest.mark.parametrize("out_dtype", [F32, BF16, F16])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_gemv_q4_types(K, dtype, out_dtype):
    packed, scale, zero = K.pack_q4(normal(1, 100, 8192), 128, True)
    x = normal(2, 2, 8192, dtype=dtype)
    got = K.gemv_q4(x, packed, scale, out_dtype=out_dtype)
    assert got.dtype == out_dtype
    assert_q4(got, x, packed, scale, zero, None)
    with pytest.raises(ValueError, match="aligned"):
        K.gemv_q4(normal(2, 2, 8196, dtype=dtype)[:, 4:], packed, scale)


def test_gemv_q4_extreme_rows(K):
    """Rows of very small, very large and mixed magnitude keep fp32's precision; NaN and infinities go through."""
    packed, scale, zero = K.pack_q4(normal(1, 70, 256), 64, False)
    x = normal(2, 4, 256)
    x[0] *= 1e-30
    x[1] *= 1e30
    x[2, ::2] *= 1e-6
    assert_q4(K.gemv_q4(x, packed, scale, zero), x, packed, scale, zero, None)
    x[3, 5] = math.nan
    got = K.gemv_q4(x, packed, scale, zero)
    assert torch.isnan(got[3]).all() and torch.isfinite(got[:3]).all()


# ------------------------------------------------- together, and how they are called
def test_one_sequence_written_token_by_token(K):
    """A prompt in two chunks, then single tokens over a rolling cache, each from 4-bit projections: against the whole
    sequence at once in 64 bits (a window of 28 keys and 4 first ones)."""
    hidden, h, kv, d, sinks, capacity = 256, 8, 2, 64, 4, 32
    window = capacity - sinks
    prompt, steps = 20, 40
    total = prompt + steps
    cos, sin = table(d, total, theta=1000000.0)
    wqkv = K.pack_q4(normal(1, (h + 2 * kv) * d, hidden), 64)
    wo = K.pack_q4(normal(2, hidden, h * d) * 0.05, 64, symmetric=False)
    x = normal(3, total, hidden, dtype=BF16)
    k_cache = torch.full((1, kv, capacity, d), math.nan, device="cuda", dtype=BF16)
    v_cache = k_cache.clone()
    got, heads_in = [], []
    done = 0
    for count in [13, 7] + [1] * steps:
        rows = K.gemv_q4(x[done : done + count], *wqkv)
        heads_in.append(rows)
        heads = rows.view(1, count, h + 2 * kv, d).transpose(1, 2)
        q = K.rope_append(heads[:, :h], heads[:, h : h + kv], heads[:, h + kv :], cos, sin, int32([done]), k_cache, v_cache,
                          sinks=sinks, layout="half")  # fmt: skip
        # the chunks of the prompt fit in the cache's slots; a single token sees every slot that is filled
        o = K.window_attention(q, k_cache, v_cache, right=0 if count > 1 else None, starts=int32([done]),
                               lengths=int32([done + count]))  # fmt: skip
        got.append(K.gemv_q4(o[0], *wo, out_dtype=F32))
        done += count
    # from the same projections on (they have their own test), every key at its own place
    heads = torch.cat(heads_in).view(1, total, h + 2 * kv, d).transpose(1, 2)
    q = K.rope(heads[:, :h], cos, sin, layout="half")
    k = K.rope(heads[:, h : h + kv], cos, sin, layout="half")
    zero = torch.zeros(1, device="cuda")
    seen = visible(total, total, zero, zero + total, window - 1, 0, sinks)
    exact, allowed = attention(q, k, heads[:, h + kv :], seen, d**-0.5)
    from text_side import unpacked

    w = unpacked(*wo)
    exact, allowed = exact.reshape(total, -1), allowed.reshape(total, -1)
    off = allowed @ w.abs().T + 60 * 2.0**-23 * (exact.abs() @ w.abs().T)
    assert torch.all((torch.cat(got).double() - exact @ w.T).abs() <= off)
    # and the rolled cache is the window over the whole sequence, in one call
    whole = K.window_attention(q, k, heads[:, h + kv :], left=window - 1, sinks=sinks)
    assert torch.all((whole.double().view(total, -1) - exact).abs() <= allowed)


def one_step(K, state):
    cos, sin, starts, heads, k_cache, v_cache, lengths, weights = state
    q = K.rope_append(heads[:, :8], heads[:, 8:10], heads[:, 10:], cos, sin, starts, k_cache, v_cache, sinks=4)
    o = K.window_attention(q, k_cache, v_cache, right=None, lengths=lengths)
    return K.gemv_q4(o.view(2, -1), *weights)


def step_state(K, seed):
    cos, sin = table(128, 4000)
    k_cache, v_cache = normal(seed, 2, 2, 1500, 128, dtype=BF16), normal(seed + 1, 2, 2, 1500, 128, dtype=BF16)
    heads = normal(seed + 2, 2, 1, 12, 128, dtype=BF16).transpose(1, 2)
    return cos, sin, int32([3000, 700]), heads, k_cache, v_cache, int32([3001, 701]), K.pack_q4(normal(7, 300, 1024), 64)


def test_captured_replayed_and_on_other_streams(K):
    """Two graphs captured one after the other and replayed in turn, with new inputs in their buffers; then the same
    calls at once on two streams: every answer that of an eager call, bit for bit."""
    states = [step_state(K, 10), step_state(K, 20)]
    expected = [one_step(K, tuple(t.clone() if isinstance(t, torch.Tensor) else t for t in s)) for s in states]
    graphs, outs = [], []
    for s in states:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(one_step(K, s))
        graphs.append(graph)
    for _ in range(3):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, e) for o, e in zip(outs, expected))
    fresh = step_state(K, 30)
    wanted = one_step(K, tuple(t.clone() if isinstance(t, torch.Tensor) else t for t in fresh))
    for mine, new in zip(states[0], fresh):
        if isinstance(mine, torch.Tensor):
            mine.copy_(new)
    graphs[0].replay()
    graphs[1].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], wanted) and torch.equal(outs[1], expected[1])
    states = [step_state(K, 10), step_state(K, 20)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(20):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i].append(one_step(K, states[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(o, expected[i]) for i in (0, 1) for o in got[i])


@pytest.mark.parametrize("n", [1, 300])
def test_same_answer_every_time(K, n):
    q, k, v = normal(1, 2, 8, n, 128, dtype=BF16), normal(2, 2, 2, 9000, 128, dtype=BF16), normal(3, 2, 2, 9000, 128, dtype=BF16)
    first = K.window_attention(q, k, v)
    assert all(torch.equal(first, K.window_attention(q, k, v)) for _ in range(5))
    w = K.pack_q4(normal(4, 500, 4096), 64)
    x = normal(5, n if n < 64 else 16, 4096, dtype=BF16)
    first = K.gemv_q4(x, *w)
    assert all(torch.equal(first, K.gemv_q4(x, *w)) for _ in range(5))


@pytest.mark.parametrize("n, n_kv, b, heads, kv", [(1, 40, 2, 8, 2), (1, 700, 1, 20, 5), (1, 20000, 1, 8, 1), (3, 90, 2, 4, 4),
                                                   (300, 300, 2, 4, 2), (257, 640, 1, 3, 3)])  # fmt: skip
def test_window_attention_onto_its_queries(K, n, n_kv, b, heads, kv):
    """In place on q's rows, in every form of the split and in whole tiles, rows that are computed again among them."""
    q = normal(1, b, n, heads, 128, dtype=BF16).transpose(1, 2)
    k, v = normal(2, b, kv, n_kv, 128, dtype=BF16), normal(3, b, kv, n_kv, 128, dtype=BF16)
    v[:, :, 5] = math.nan
    for left in (None, 20):
        expected = K.window_attention(q, k, v, left=left)
        own = q.transpose(1, 2).contiguous().transpose(1, 2)
        rows = own.transpose(1, 2).view(b, n, heads * 128)
        assert K.window_attention(own, k, v, left=left, out=rows) is rows
        assert torch.equal(rows.view(torch.int16), expected.view(torch.int16))


def test_outputs_whose_rows_overlap_are_refused(K):
    cos, sin = table(64, 9)
    x = normal(1, 2, 4, 3, 64)
    room = torch.zeros(4096, device="cuda")
    for strides in [(768, 192, 32, 1), (192, 192, 64, 1), (768, 64, 64, 1)]:
        with pytest.raises(ValueError, match="overlap"):
            K.rope(x, cos, sin, out=room.as_strided((2, 4, 3, 64), strides))
    q, k = x.bfloat16(), normal(2, 2, 2, 3, 64, dtype=BF16)
    with pytest.raises(ValueError, match="overlap"):
        K.window_attention(q, k, k, out=room.bfloat16().as_strided((2, 3, 256), (768, 64, 1)))


def test_rolling_append_past_the_tables(K):
    """Tokens whose position has no table row are not appended, and take no slot from those before them."""
    cos, sin = table(64, 14)
    q, k, v = packed_heads(4, 2, 8, 2, 1, 64, BF16)
    k_cache, v_cache = torch.zeros(2, 1, 6, 64, device="cuda", dtype=BF16), torch.zeros(2, 1, 6, 64, device="cuda", dtype=BF16)
    K.device_error()
    K.rope_append(q, k, v, cos, sin, int32([10, 3]), k_cache, v_cache, sinks=2)
    assert K.device_error() & ERR_BAD_ARGUMENT
    for s, first in ((0, 10), (1, 3)):
        latest = {2 + (p - 2) % 4: p for p in range(max(first, 2), min(first + 8, 14))}  # positions 10 to 13; 7 to 10
        assert len(latest) == 4
        for slot, p in latest.items():
            assert torch.equal(v_cache[s, :, slot], v[s, :, p - first])
            assert_turned(k_cache[s, :, slot], k[s, :, p - first], cos[p], sin[p], "interleaved")
        assert torch.all(v_cache[s, :, :2] == 0)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim, rotary", [(64, 64), (128, 32), (80, 40), (10, 2)])
def test_rows_outside_the_tables_are_nan_in_every_column(K, dtype, layout, dim, rotary):
    cos, sin = table(rotary, 8)
    q, k, v = packed_heads(3, 2, 4, 5, 2, dim, dtype)
    K.device_error()
    got = K.rope(q, cos, sin, torch.tensor([3, -1, 7, 8], device="cuda"), layout=layout)
    assert K.device_error() & ERR_BAD_ARGUMENT
    assert torch.isnan(got[:, :, [1, 3]]).all()
    at = torch.tensor([3, 7], device="cuda")
    assert_turned(got[:, :, [0, 2]], q[:, :, [0, 2]], cos[at], sin[at], layout)
    caches = torch.zeros(2, 2, 2, 8, dim, device="cuda", dtype=dtype)
    got = K.rope_append(q, k, v, cos, sin, int32([6, -2]), *caches, layout=layout)
    assert torch.isnan(got[0, :, 2:]).all() and torch.isnan(got[1, :, :2]).all()
    assert torch.isfinite(got[0, :, :2]).all() and torch.isfinite(got[1, :, 2:]).all() and torch.isfinite(caches).all()
    assert torch.equal(caches[1, 0, :, 6:], v[0, :, :2]) and torch.all(caches[:, 0, :, :6] == 0)
    assert torch.equal(caches[1, 1, :, :2], v[1, :, 2:]) and torch.all(caches[:, 1, :, 2:] == 0)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_gemv_q4_zero_points(K, dtype, group):
    """Every zero point of 4 bits; one beyond them marks its weight row alone and the device error word."""
    n, k = 200, 6 * group + 128
    packed, scale, _ = K.pack_q4(normal(1, n, k), group)
    zero = (torch.arange(n * scale.shape[1], device="cuda") % 16).to(torch.uint8).view_as(scale)
    x = normal(2, 3, k, dtype=dtype)
    K.device_error()
    good = K.gemv_q4(x, packed, scale, zero)
    assert_q4(good, x, packed, scale, zero, None)
    assert K.device_error() == 0
    rows = torch.tensor([0, 37, 130, 199], device="cuda")
    for row, value in zip(rows.tolist(), (16, 17, 128, 255)):
        zero[row, row % scale.shape[1]] = value
    got = K.gemv_q4(x, packed, scale, zero)
    assert K.device_error() & ERR_BAD_ARGUMENT
    assert torch.isnan(got[:, rows]).all()
    rest = torch.ones(n, dtype=torch.bool, device="cuda").index_fill(0, rows, False)
    assert torch.equal(got[:, rest], good[:, rest])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("m, n, k", [(1, 130, 2560), (2, 300, 256), (20, 70, 1280)])
def test_gemv_q4_rows_near_the_end_of_the_range(K, dtype, group, m, n, k):
    """Unscaled group sums beyond fp32, finite results: weights of one sign and x of 2e36 to 8e36."""
    w = normal(1, n, k).abs() * 1e-4
    packed, scale, zero = K.pack_q4(w, group, False)
    x = ((0.2 + 0.8 * torch.rand(m, k, device="cuda", generator=torch.Generator("cuda").manual_seed(m))) * 8e36).to(dtype)
    if m > 1:
        x[m // 2] *= 1e-36  # a row of ordinary size beside them
    bias = normal(3, n)
    got = K.gemv_q4(x, packed, scale, zero, bias, out_dtype=F32)
    assert torch.isfinite(got).all()
    assert_q4(got, x, packed, scale, zero, bias)
    x[0, 5] = math.inf
    assert not torch.isfinite(K.gemv_q4(x, packed, scale, zero, bias)[0]).any()  # inf, or NaN from a weight of 0


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n, n_kv, heads, kv", [(1, 40, 2, 1), (1, 700, 20, 5), (1, 20000, 8, 1), (3, 90, 4, 4), (300, 300, 4, 2)])
def test_values_near_the_end_of_the_range(K, dim, n, n_kv, heads, kv):
    """Values of 1e38 to 3e38: their weighted sum leaves fp32, their mean does not; and scores whose unscaled sums do."""
    gen = torch.Generator("cuda").manual_seed(n_kv)
    q, k = normal(1, 1, heads, n, dim, dtype=BF16), normal(2, 1, kv, n_kv, dim, dtype=BF16)
    v = ((1 + 2 * torch.rand(1, kv, n_kv, dim, device="cuda", generator=gen)) * 1e38).to(BF16)
    v[..., ::3] *= -1e-38  # ordinary values beside them
    for left in (None, 30):
        got = K.window_attention(q, k, v, left=left)
        assert torch.isfinite(got).all()
        assert_attends(got, q, k, v, left=left)
    big = torch.full_like(q, 2.0**62)
    k = torch.where(torch.arange(n_kv, device="cuda")[:, None] % 7 == 0, 2.0**62, -(2.0**62)).to(BF16).expand(1, kv, n_kv, dim).contiguous()
    v = normal(3, 1, kv, n_kv, dim, dtype=BF16)
    # scores of +- dim 2^124 (2^130 or 2^131 unscaled): the keys of the larger one share the row
    got = K.window_attention(big, k, v, right=None, scale=2.0**-10)
    mean = v[:, :, ::7].double().mean(dim=2, keepdim=True).repeat_interleave(heads // kv, dim=1).expand(1, heads, n, dim)
    off = (got.double().view(1, n, heads, dim).transpose(1, 2) - mean).abs()
    assert torch.all(off <= 2.0**-8 * mean.abs() + (n_kv + 8) * 2.0**-23 * v.double().abs().amax())


@pytest.mark.parametrize("n, n_kv", [(1, 60), (5, 60), (40, 2000), (200, 500), (10, 4), (300, 100)])
def test_positions_by_default_count_from_the_last_key(K, n, n_kv):
    """Without `starts` the last query is at the last key, whatever `lengths` say: a chunk over a partly filled cache needs
    its starts. With more queries than keys the first ones see nothing."""
    q = normal(1, 3, 4, n, 64, dtype=BF16)
    k, v = normal(2, 3, 2, n_kv, 64, dtype=BF16), normal(3, 3, 2, n_kv, 64, dtype=BF16)
    lengths = int32([n_kv, max(1, n_kv // 2), max(0, n_kv - 3)])
    for left, right in [(None, 0), (20, 0), (20, 3), (None, None)]:
        got = K.window_attention(q, k, v, left=left, right=right, lengths=lengths)
        assert_attends(got, q, k, v, left=left, right=right, lengths=lengths)
        assert torch.equal(got, K.window_attention(q, k, v, left=left, right=right, lengths=lengths, starts=int32([n_kv - n] * 3)))
        if n > n_kv and right == 0:
            assert torch.all(got[:, : n - n_kv] == 0)


def test_captured_with_streams_that_fork_and_join(K):
    """Calls that each wait for two others, on several streams inside one capture; the predecessors of a call in its
    stream are a kernel, a copy and a fill in turn."""
    w = K.pack_q4(normal(7, 12 * 128, 256), 64)
    out = K.pack_q4(normal(8, 200, 1024), 128)
    cos, sin = table(128, 4000)
    x, caches = normal(1, 2, 256, dtype=BF16), normal(2, 2, 2, 2, 1500, 128, dtype=BF16)
    starts, lengths, room = int32([3000, 700]), int32([3001, 701]), torch.empty(2, 256, device="cuda", dtype=BF16)

    def step(x, caches, side):
        main = torch.cuda.current_stream()
        room.copy_(x)
        heads = K.gemv_q4(room, *w).view(2, 1, 12, 128).transpose(1, 2)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            turned = K.rope(heads[:, :8], cos, sin, starts[:, None].contiguous())
        q = K.rope_append(heads[:, :8], heads[:, 8:10], heads[:, 10:], cos, sin, starts, caches[0], caches[1], sinks=4)
        main.wait_stream(side)
        o = K.window_attention(q, caches[0], caches[1], right=None, lengths=lengths)
        o = o + K.window_attention(turned, caches[0], caches[1], right=None, lengths=lengths)
        room.zero_()
        return K.gemv_q4(o.view(2, -1), *out), q, turned

    side = torch.cuda.Stream()
    expected = step(x, caches.clone(), side)
    assert torch.equal(expected[1], expected[2])
    held = caches.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(x, held, side)
    for _ in range(5):
        held.copy_(caches)
        for t in got:
            t.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, expected))
