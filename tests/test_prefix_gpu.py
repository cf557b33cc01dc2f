"""Attention behind a shared prefix on a B200 against its definition in 64 bits, each
element within what its roundings allow."""

import math

import pytest
import torch

from batch_side import assert_i8, assert_prefix, quantized
from text_side import assert_attends, assert_turned

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def K():
    from iris_b200 import kernels

    return kernels


def normal(seed, *shape, dtype=BF16):
    return torch.randn(*shape, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)).to(dtype)


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def inputs(seed, b, g, h, kv, n, p, m, d, dtype=BF16):
    q = normal(seed, b, n, (h + 2) * d, dtype=dtype).view(b, n, h + 2, d).transpose(1, 2)[:, :h]
    pk, pv = normal(seed + 1, 2, g, kv, p, d, dtype=dtype)
    k, v = normal(seed + 2, 2, b, kv, m, d, dtype=dtype)
    return q, pk, pv, k, v


def ragged(seed, b, lo, hi):
    gen = torch.Generator().manual_seed(seed)
    return torch.randint(lo, hi + 1, (b,), generator=gen, dtype=torch.int32).cuda()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("b, g, h, kv", [(1, 1, 1, 1), (3, 1, 4, 2), (4, 2, 5, 5), (6, 3, 20, 5), (2, 2, 8, 1), (16, 1, 16, 2), (5, 1, 21, 3)])
def test_single_tokens(K, dim, dtype, b, g, h, kv):
    for p, m in [(1, 1), (63, 2), (64, 16), (65, 17), (300, 64), (1023, 130), (2100, 513)]:
        x = inputs(p + m, b, g, h, kv, 1, p, m, dim, dtype)
        lengths = ragged(p, b, 1, m)
        got = K.prefix_attention(*x, starts=lengths - 1, lengths=lengths)
        assert got.shape == (b, 1, h * dim) and got.dtype == dtype
        assert_prefix(got, *x, starts=lengths - 1, lengths=lengths)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("b, g, h, kv", [(1, 1, 3, 1), (4, 2, 4, 2), (9, 3, 5, 5), (2, 1, 20, 5)])
@pytest.mark.parametrize("n", [2, 5, 16, 31, 70, 128, 129, 300])
def test_chunks_and_prompts(K, dim, b, g, h, kv, n):
    for (p, extra), right in zip([(1, 0), (64, 1), (129, 40), (700, 200)], [0, None, 0, 3]):
        m = n + extra
        x = inputs(p + n, b, g, h, kv, n, p, m, dim, F16 if n % 2 else BF16)
        prefix_lengths = ragged(n, g, 0, p)
        lengths = ragged(p, b, n, m)
        got = K.prefix_attention(*x, prefix_lengths=prefix_lengths, starts=lengths - n, lengths=lengths, right=right)
        assert_prefix(got, *x, prefix_lengths=prefix_lengths, starts=lengths - n, lengths=lengths, right=right)


@pytest.mark.parametrize("b, g, h, kv, n, p, m", [
    (64, 1, 8, 1, 1, 5000, 300),  # many rows of one key head over a long prefix
    (40, 2, 12, 4, 1, 9000, 1100),
    (3, 1, 4, 4, 400, 3000, 500),
    (1, 1, 8, 2, 64, 20000, 64),  # a chunk over a long prefix
    (2, 1, 2, 2, 1024, 4096, 1024),
    (7, 1, 48, 8, 3, 77, 1500),
    (33, 1, 1, 1, 1, 12345, 1),
    (1, 1, 32, 8, 1, 40000, 3000),
])  # fmt: skip
def test_long(K, b, g, h, kv, n, p, m):
    for dim in (64, 128):
        x = inputs(p, b, g, h, kv, n, p, m, dim)
        lengths = ragged(p, b, n, m)
        got = K.prefix_attention(*x, starts=lengths - n, lengths=lengths)
        assert_prefix(got, *x, starts=lengths - n, lengths=lengths)


@pytest.mark.parametrize("n", [1, 4, 40, 200])
def test_lengths_at_their_ends(K, n):
    """Prefixes and caches that are empty, out of range or unseen; rows that see nothing are 0."""
    b, g, h, kv, p, m, d = 6, 3, 4, 2, 200, 250, 64
    x = inputs(n, b, g, h, kv, n, p, m, d)
    for prefix_lengths, lengths, starts in [
        ([0, 0, 0], [0] * 6, [0] * 6),
        ([0, 200, 0], [0, 1, 0, 1, 250, 9], [0, 0, -300, -300, -n, 5]),
        ([-7, 900, 64], [-1, 900, 1, 64, 65, 128], [3, 100000, 2**31 - 1, -(2**31), 0, -1]),
        ([1, 63, 65], [250] * 6, [-5, -n + 1, 0, 3, 250, 249]),
    ]:
        kw = dict(prefix_lengths=int32(prefix_lengths), lengths=int32(lengths), starts=int32(starts))
        for right in (0, 2, None):
            got = K.prefix_attention(*x, right=right, **kw)
            assert_prefix(got, *x, right=right, **kw)
            if prefix_lengths == [0, 0, 0]:
                assert torch.equal(got, torch.zeros_like(got))
    got = K.prefix_attention(*x)  # no lengths: all of them, the tokens at the end
    if n <= m:
        assert_prefix(got, *x)
    q, pk, pv, k, v = x
    assert_prefix(K.prefix_attention(q, pk[:, :, :0], pv[:, :, :0], k, v), q, pk[:, :, :0], pv[:, :, :0], k, v)
    assert_prefix(K.prefix_attention(q, pk, pv, k[:, :, :0], v[:, :, :0]), q, pk, pv, k[:, :, :0], v[:, :, :0])
    none = K.prefix_attention(q, pk[:, :, :0], pv[:, :, :0], k[:, :, :0], v[:, :, :0])
    assert torch.equal(none, torch.zeros_like(none))
    assert K.prefix_attention(q[:, :, :0], pk, pv, k, v).shape == (b, 0, h * d)
    assert K.prefix_attention(q[:0], pk, pv, k[:0], v[:0]).shape == (0, n, h * d)


@pytest.mark.parametrize("n", [1, 3, 40, 160])
@pytest.mark.parametrize("dim", [64, 128])
def test_what_lies_in_hidden_places_takes_no_part(K, n, dim):
    b, g, h, kv, p, m = 4, 2, 6, 2, 330, n + 100
    q, pk, pv, k, v = inputs(n, b, g, h, kv, n, p, m, dim)
    prefix_lengths, lengths = int32([101, 320]), int32([n, n + 7, n + 64, n + 99])
    kw = dict(prefix_lengths=prefix_lengths, lengths=lengths, starts=lengths - n)
    want = K.prefix_attention(q, pk, pv, k, v, **kw)
    for bad in (math.nan, math.inf, -math.inf):
        dirty = [t.clone() for t in (pk, pv, k, v)]
        for t in dirty[:2]:
            for i, length in enumerate(prefix_lengths.tolist()):
                t[i, :, length:] = bad
        for t in dirty[2:]:
            for i, length in enumerate(lengths.tolist()):
                t[i, :, length:] = bad
        assert torch.equal(K.prefix_attention(q, *dirty, **kw), want)
    if n > 1:  # a key that some rows of a tile see and others do not
        dirty = [pk, pv, k.clone(), v.clone()]
        dirty[2][:, :, lengths[0] - 1], dirty[3][:, :, lengths[0] - 1] = math.nan, math.nan
        got = K.prefix_attention(q, *dirty, **kw)
        assert_prefix(got[:1, : n - 1], q[:1, :, : n - 1], pk[:1], pv[:1], k[:1], v[:1], prefix_lengths=prefix_lengths[:1],
                      starts=lengths[:1] - n, lengths=lengths[:1])  # fmt: skip
        assert bool(got[0, n - 1].isnan().all())


@pytest.mark.parametrize("n, p", [(1, 700), (6, 100), (140, 300)])
def test_visible_values_that_are_not_finite(K, n, p):
    """NaN and infinities that a row sees reach it as the formula has it."""
    q, pk, pv, k, v = inputs(n, 4, 1, 4, 2, n, p, n, 64)
    pv[0, 0, 5, 3], pv[0, 1, 7, 1], v[2, 1, 0, 9] = math.inf, math.nan, -math.inf
    pk[0, 0, 9] = 0
    got = K.prefix_attention(q, pk, pv, k, v).view(4, n, 4, 64)
    assert bool(got[:, :, :2, 3].isposinf().all()) and bool(got[:, :, 2:, 1].isnan().all()) and bool(got[2, :, 2:, 9].isneginf().all())
    got[:, :, :2, 3] = got[:, :, 2:, 1] = got[2, :, 2:, 9] = 0
    assert bool(got.isfinite().all())
    pk[0, :, :] = math.nan
    assert bool(K.prefix_attention(q, pk, pv, k, v).isnan().all())


@pytest.mark.parametrize("n, p", [(1, 900), (7, 300), (150, 200)])
def test_values_and_scores_near_the_end_of_the_types(K, n, p):
    for dtype in (BF16, F16):
        q, pk, pv, k, v = inputs(n, 3, 1, 4, 2, n, p, n + 20, 128, dtype)
        big = torch.finfo(dtype).max
        v, pv = v.sign() * big * 0.9, pv.sign() * big * 0.9
        assert_prefix(K.prefix_attention(q, pk, pv, k, v), q, pk, pv, k, v)
        same = torch.full_like(v, big), torch.full_like(pv, big)
        got = K.prefix_attention(q, pk, same[1], k, same[0])
        assert bool((got.float() >= big * (1 - 2.0**-7)).all())
        # far scores: one key takes all the weight
        got = K.prefix_attention(q * 30, pk, pv.sign(), k * 30, v.sign())
        assert_prefix(got, q * 30, pk, pv.sign(), k * 30, v.sign())
    q, pk, pv, k, v = inputs(n, 3, 1, 4, 2, n, p, n + 20, 128)
    for scale in (1e-30, 0.5, 3.0):
        assert_prefix(K.prefix_attention(q, pk, pv, k, v, scale=scale), q, pk, pv, k, v, scale=scale)


@pytest.mark.parametrize("n", [1, 9, 200])
def test_strides_expanded_heads_and_outputs(K, n):
    b, h, kv, p, m, d = 4, 6, 3, 140, n + 30, 64
    q, pk, pv, k, v = inputs(n, b, 2, h, kv, n, p, m, d)
    want = K.prefix_attention(q, pk, pv, k, v)
    assert_prefix(want, q, pk, pv, k, v)
    # token-major caches, wider rows, an expanded group / head / sample
    major = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (pk, pv, k, v)]
    assert torch.equal(K.prefix_attention(q, *major), want)
    wide = [torch.cat([t, t], dim=-1)[..., :d] for t in (pk, pv, k, v)]
    assert torch.equal(K.prefix_attention(q.contiguous(), *wide), want)
    assert torch.equal(K.prefix_attention(q, pk[:1].expand(2, -1, -1, -1), pv[:1].expand(2, -1, -1, -1), k, v)[:2], want[:2])
    one = [t[:, :1].expand(-1, kv, -1, -1) for t in (pk, pv, k, v)]
    assert torch.equal(K.prefix_attention(q, *one), K.prefix_attention(q, *(t.contiguous() for t in one)))
    all_samples = [pk, pv, k[:1].expand(b, -1, -1, -1), v[:1].expand(b, -1, -1, -1)]
    assert torch.equal(K.prefix_attention(q, *all_samples), K.prefix_attention(q, *(t.contiguous() for t in all_samples)))
    # outputs: rows of a wider buffer whose other columns stay, and q's own rows
    room = torch.full((b, n, h * d + 64), 7.0, device="cuda", dtype=BF16)
    assert K.prefix_attention(q, pk, pv, k, v, out=room[..., 32 : 32 + h * d]).data_ptr() == room.data_ptr() + 64
    assert torch.equal(room[..., 32 : 32 + h * d], want) and bool((room[..., :32] == 7).all()) and bool((room[..., 32 + h * d :] == 7).all())
    rows = q.transpose(1, 2).contiguous()
    K.prefix_attention(rows.transpose(1, 2), pk, pv, k, v, out=rows.view(b, n, h * d))
    assert torch.equal(rows.view(b, n, h * d), want)


def test_in_place_rows_that_are_computed_again(K):
    """Onto q's own rows where some are not finite at first (a hidden NaN): they are read before they are written."""
    b, h, n, p, d = 3, 4, 150, 90, 128
    q, pk, pv, k, v = inputs(5, b, 1, h, 2, n, p, n, d)
    want = K.prefix_attention(q, pk, pv, k, v)
    v = v.clone()
    v[:, :, n - 1] = math.nan  # seen by the last row alone
    rows = q.transpose(1, 2).contiguous()
    K.prefix_attention(rows.transpose(1, 2), pk, pv, k, v, out=rows.view(b, n, h * d))
    got = rows.view(b, n, h * d)
    clean = inputs(5, b, 1, h, 2, n, p, n, d)
    assert_prefix(got[:, : n - 1], clean[0][:, :, : n - 1], pk, pv, clean[3], clean[4], starts=int32([0] * b))
    assert bool(got[:, n - 1].isnan().all()) and bool(want.isfinite().all())


@pytest.mark.parametrize("n", [1, 150])
def test_offsets_past_32_bits(K, n):
    """Token strides that put the last keys past 2^31 elements and 2^32 bytes."""
    p, d, stride = 140, 64, 2**24 + 8
    room = torch.zeros(p * stride, device="cuda", dtype=BF16)
    q, pk, pv, k, v = inputs(6, 2, 1, 2, 1, n, p, p, d)
    far = [room[i * 64 :].as_strided((1, 1, p, d), (0, 0, stride, 1)) for i in range(4)]
    far[0].copy_(pk)
    far[1].copy_(pv)
    far[2].copy_(k[:1])
    far[3].copy_(v[:1])
    k, v = k[:1].expand(2, -1, -1, -1), v[:1].expand(2, -1, -1, -1)
    got = K.prefix_attention(q, far[0], far[1], far[2].expand(2, -1, -1, -1), far[3].expand(2, -1, -1, -1), starts=int32([0, 70]))
    assert_prefix(got, q, pk, pv, k, v, starts=int32([0, 70]))


def test_like_one_attention_over_all_keys(K):
    for n, m in [(1, 40), (30, 64), (200, 200)]:
        q, pk, pv, k, v = inputs(n, 3, 1, 8, 2, n, 333, m, 128)
        keys = torch.cat([pk.expand(3, -1, -1, -1), k], dim=2), torch.cat([pv.expand(3, -1, -1, -1), v], dim=2)
        assert_attends(K.prefix_attention(q, pk, pv, k, v), q, *keys)
        assert_prefix(K.window_attention(q, *keys), q, pk, pv, k, v)


def test_the_same_results_each_time(K):
    for n in (1, 5, 140):
        x = inputs(n, 8, 2, 8, 2, n, 3000, n + 300, 128)
        want = K.prefix_attention(*x)
        for _ in range(5):
            assert torch.equal(K.prefix_attention(*x), want)


def test_streams_graphs_and_written_just_before(K):
    sets = [inputs(20 + i, 8, 1, 8, 2, 2, 1500, 90, 128) for i in range(2)]
    lengths = [ragged(i, 8, 2, 90) for i in range(2)]
    want = [K.prefix_attention(*x, starts=n - 2, lengths=n) for x, n in zip(sets, lengths)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(K.prefix_attention(*sets[i], starts=lengths[i] - 2, lengths=lengths[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])
    held, n = [t.clone(memory_format=torch.contiguous_format) for t in sets[0]], lengths[0].clone()
    starts = n - 2
    for turn in range(20):  # every input is written by the kernel before, and again by the one behind
        i = turn & 1
        for t, s in zip(held, sets[i]):
            t.copy_(s)
        n.copy_(lengths[i])
        starts.copy_(lengths[i] - 2)
        out = K.prefix_attention(*held, starts=starts, lengths=n)
        for t in held:
            t.fill_(math.nan)
        assert torch.equal(out, want[i])
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(K.prefix_attention(*held, starts=starts, lengths=n))
        graphs.append(graph)
    for i in (1, 0, 1):
        for t, s in zip(held, sets[i]):
            t.copy_(s)
        n.copy_(lengths[i])
        starts.copy_(lengths[i] - 2)
        torch.cuda.synchronize()
        for stream, graph in zip(streams, graphs):  # side by side
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want[i]) for o in outs)


def test_a_layers_step(K):
    """A step of a batch behind one instruction, as it is used: 8-bit projection, append, attention, 8-bit projection."""
    from iris_b200.tables import rope_table

    b, h, kv, d, p, room, width = 12, 20, 5, 128, 700, 64, 2560
    cos, sin = rope_table(d, 1000, device="cuda")
    w_qkv = K.quantize_i8(normal(1, (h + 2 * kv) * d, width, dtype=torch.float32) * 0.02)
    w_out = K.quantize_i8(normal(2, width, h * d, dtype=torch.float32) * 0.02)
    pk, pv = normal(3, 2, 1, kv, p, d)
    k_cache, v_cache = normal(4, 2, b, kv, room, d)
    positions = ragged(5, b, 0, room - 4)
    for turn in range(3):
        x = normal(6 + turn, b, width)
        rows = K.gemm_i8(x, *w_qkv)
        assert_i8(rows, *quantized(x), *w_qkv)
        heads = rows.view(b, 1, h + 2 * kv, d).transpose(1, 2)
        # rotary positions count the prefix, slots of the caches do not: the tables from row p on
        before = k_cache.clone()
        q = K.rope_append(heads[:, :h], heads[:, h : h + kv], heads[:, h + kv :], cos[p:], sin[p:], positions, k_cache, v_cache,
                          layout="half")  # fmt: skip
        at = (positions + p).long()[:, None, None]
        assert_turned(q, heads[:, :h], cos[at], sin[at], "half")
        assert int((before != k_cache).any(-1).sum()) == b * kv
        o = K.prefix_attention(q, pk, pv, k_cache, v_cache, starts=positions, lengths=positions + 1)
        assert_prefix(o, q, pk, pv, k_cache, v_cache, starts=positions, lengths=positions + 1)
        y = K.gemm_i8(o[:, 0], *w_out)
        assert_i8(y, *quantized(o[:, 0]), *w_out)
        positions = positions + 1


def test_behind_one_another(K):
    """Kernels with TMEM of different sizes in a chain, each starting while the one before ends."""
    b, n, h, kv, d = 4, 300, 20, 5, 64
    q, pk, pv, k, v = inputs(40, b, 1, h, kv, n, 500, n, d)
    one = inputs(41, 16, 2, 8, 2, 1, 2000, 90, d)
    packed, scale = K.quantize_i8(normal(42, 700, h * d, dtype=torch.float32))
    many, many_scale = K.quantize_i8(normal(43, 2600, 900, dtype=torch.float32))
    x8, x_scale = K.quantize_i8(normal(44, 16, h * d))
    y8, y_scale = K.quantize_i8(normal(45, 600, 900))

    def chain():
        a = K.window_attention(q, k, v)
        first = K.gemm_i8(x8, packed, scale, x_scale=x_scale)
        p = K.prefix_attention(q, pk, pv, k, v)
        second = K.gemm_i8(p.view(b * n, h * d)[:40], packed, scale)
        t = K.prefix_attention(*one)
        third = K.gemm_i8(y8, many, many_scale, x_scale=y_scale)
        w = K.window_attention(q, k, v, left=100)
        last = K.gemm_i8(w.view(b * n, h * d)[:1], packed, scale)
        return a, first, p, second, t, third, w, last

    want = chain()
    assert_attends(want[0], q, k, v)
    assert_prefix(want[2], q, pk, pv, k, v)
    assert_i8(want[5], y8, y_scale, many, many_scale)
    torch.cuda.synchronize()
    for _ in range(60):
        for got, x in zip(chain(), want):
            assert torch.equal(got, x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = [chain() for _ in range(3)]
    for _ in range(20):
        graph.replay()
    assert all(torch.equal(got, x) for outs in held for got, x in zip(outs, want))


@pytest.mark.parametrize("n, p", [(1, 300), (3, 77), (150, 300), (1, 0)])
def test_the_stride_of_a_lone_token_is_not_read(K, n, p):
    """Through the C ABI, where any value may stand in it."""
    import ctypes

    from iris_b200 import _lib
    from test_prefix import PREFIX

    lib, d = _lib.load(), 64
    q, pk, pv, k, v = inputs(50, 2, 1, 4, 2, n, p, 1, d)
    starts = int32([n, n])  # the one key is seen by every row
    want = K.prefix_attention(q, pk, pv, k, v, starts=starts)
    assert_prefix(want, q, pk, pv, k, v, starts=starts)
    for stride in (0, -8, -(1 << 20), 1 << 34, 1 << 45):
        def rows(t, n_stride=None):
            return t.data_ptr(), t.stride(0), t.stride(1), t.stride(2) if n_stride is None else n_stride

        out = torch.full_like(want, 7.0)

        def problem(workspace=0, room=0):
            return PREFIX.pack(*rows(q), *rows(pk), *rows(pv), *rows(k, stride), *rows(v, -stride), out.data_ptr(), n * 4 * d, 4 * d, 0,
                               starts.data_ptr(), 0, workspace, room, 1, 2, 1, 4, 2, n, p, 1, d, 0, d**-0.5)  # fmt: skip

        need = ctypes.c_int64(-1)
        assert lib.iris_prefix_attn_workspace(problem(), ctypes.byref(need)) == 0
        workspace = torch.empty(max(need.value, 16), device="cuda", dtype=torch.uint8)
        stream = torch.cuda.current_stream().cuda_stream
        assert lib.iris_prefix_attn_fwd(problem(workspace.data_ptr(), need.value), stream) == 0
        torch.cuda.synchronize()
        assert torch.equal(out, want)
