"""The 8-bit linear on a B200: rows to 8 bits (bit for bit) and the product."""

import math

import pytest
import torch

from batch_side import assert_i8, quantized
from text_side import HALF_STEP

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def K():
    from iris_b200 import kernels

    return kernels


def rows(seed, m, k, dtype=torch.bfloat16, spread=True):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(m, k, device="cuda", generator=gen)
    return (x * torch.exp(torch.randn(k, device="cuda", generator=gen)) if spread else x).to(dtype)


def assert_quantized(K, x):
    q, scale = K.quantize_i8(x)
    want, want_scale = quantized(x)
    assert q.dtype == torch.int8 and q.shape == x.shape and (x.shape[0] <= 1 or q.stride(0) % 16 == 0)
    assert torch.equal(q.double(), want)
    assert torch.equal(scale.view(torch.int32)[~scale.isnan()], want_scale.view(torch.int32)[~want_scale.isnan()])
    assert torch.equal(scale.isnan(), want_scale.isnan())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", [1, 2, 7, 8, 9, 31, 128, 509, 512, 513, 1024, 1025, 2049, 4096, 4100, 8192, 8201, 20011])
def test_rows_to_8_bits(K, dtype, k):
    for m in (1, 2, 5, 130):
        assert_quantized(K, rows(k + m, m, k, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_to_8_bits_strides(K, dtype):
    base = rows(1, 9, 700, dtype)
    for view in (base[:, :128], base[:, 3:300], base[1::2, 8:600], base[:1, 5:6], base[:, 1:]):
        assert_quantized(K, view)
    flat = rows(2, 1, 5000, dtype)[0]
    assert_quantized(K, flat[1:4001].view(8, 500))  # rows that start anywhere
    assert_quantized(K, base[:1].expand(4, 700))


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_to_8_bits_at_halves(K, dtype):
    """Quotients that are a half, or next to one: every magnitude over every largest one of a short mantissa."""
    tops = torch.arange(128, 256, device="cuda", dtype=torch.float32) / 64
    x = (torch.arange(-255, 256, device="cuda", dtype=torch.float32) / 64).expand(128, 511).clone()
    x = torch.where(x.abs() <= tops[:, None], x, 0.0)
    x = torch.cat([x, tops[:, None], -tops[:, None] / 2, tops[:, None] / 127, tops[:, None] * 1.5 / 127], dim=1).to(dtype)
    assert_quantized(K, x)
    if dtype == torch.float32:  # neighbours of the halves, a bit to either side
        h = (torch.arange(-127, 127, device="cuda", dtype=torch.float64) + 0.5) / 127
        x = (h[None] * rows(3, 64, 1, dtype).abs().double()).float()
        x = torch.cat([x, x.nextafter(torch.full_like(x, math.inf)), x.nextafter(torch.full_like(x, -math.inf))], dim=1)
        x = torch.cat([x, rows(3, 64, 1, dtype).abs()], dim=1)
        assert_quantized(K, x)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_to_8_bits_extremes(K, dtype):
    info = torch.finfo(dtype)
    x = rows(4, 12, 300, dtype)
    x[0] = 0
    x[1, 7], x[2, 0], x[3, 299] = math.inf, -math.inf, math.nan
    x[4] = info.max
    x[5, 11] = info.max
    x[6] *= info.smallest_normal
    x[7] = 0
    x[7, 5], x[7, 6] = info.smallest_normal * info.eps, -info.smallest_normal * info.eps * 3  # subnormal
    x[8] = -0.0
    x[9] = rows(5, 1, 300, torch.float32)[0].mul(1e-36).to(dtype)
    x[10, :] = info.tiny
    assert_quantized(K, x)


def product(seed, m, n, k, dtype, bias=True, out_dtype=None):
    x, w = rows(seed, m, k, dtype), rows(seed + 1, n, k, torch.float32, False)
    gen = torch.Generator(device="cuda").manual_seed(seed + 2)
    return x, w, torch.randn(n, device="cuda", generator=gen) if bias else None


def check(K, m, n, k, dtype, bias=True, out_dtype=None, seed=0):
    x, w, b = product(seed, m, n, k, dtype, bias)
    packed, scale = K.quantize_i8(w)
    want = quantized(x)
    got = K.gemm_i8(x, packed, scale, b, out_dtype=out_dtype)
    assert got.shape == (m, n) and got.dtype == (out_dtype or dtype) and got.is_contiguous()
    assert_i8(got, *want, packed, scale, b)
    q, x_scale = K.quantize_i8(x)
    again = K.gemm_i8(q, packed, scale, b, x_scale=x_scale, out_dtype=out_dtype or dtype)
    assert torch.equal(got, again)  # the same rows, quantised here or there


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 32, 33, 64, 65, 128, 129, 255, 256, 257, 300, 520, 1000])
@pytest.mark.parametrize("n, k", [(1, 1), (17, 15), (127, 128), (128, 129), (129, 1000), (300, 2560)])
def test_product_sizes(K, m, n, k):
    check(K, m, n, k, torch.bfloat16, bias=m % 2 == 1, seed=m)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("out_dtype", [None, *DTYPES])
def test_product_types(K, dtype, out_dtype):
    for m, n, k in [(1, 2561, 700), (37, 515, 6845), (200, 259, 333), (700, 770, 1301)]:
        check(K, m, n, k, dtype, out_dtype=out_dtype, seed=m)


@pytest.mark.parametrize("m", [1, 40, 300, 2048])
def test_product_wide(K, m):
    for n, k in [(2560, 2560), (5001, 4096), (256, 20000)]:
        check(K, m, n, k, torch.bfloat16, bias=False, seed=m)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 8, 9, 15, 16, 17, 31, 32, 33, 64, 65, 100, 128])
def test_a_few_rows_that_the_product_rounds(K, m, dtype):
    """Against the same rows quantised before: bit for bit, in each number of parts of K, extreme rows among them."""
    for k in (1, 7, 8, 127, 128, 129, 520, 1000, 1280, 2560, 10240 // m):
        x = rows(k, m, k, dtype)
        if m > 4:
            x[0], x[1] = 0, x[1] * torch.finfo(dtype).smallest_normal * 2.0**9
            x[2, k // 2], x[3, 0], x[4, -1] = math.inf, math.nan, torch.finfo(dtype).max
        for n in (1, 130, 2561):
            packed, scale = K.quantize_i8(rows(n, n, k, torch.float32, False))
            q, x_scale = K.quantize_i8(x)
            want = K.gemm_i8(q, packed, scale, x_scale=x_scale, out_dtype=dtype)
            for view in (x, torch.cat([x, x], dim=1)[:, :k], torch.cat([x[:, :1], x], dim=1)[:, 1:]):  # rows anywhere
                got = K.gemm_i8(view, packed, scale)
                assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0)) and torch.equal(got.isnan(), want.isnan())


def test_longest_sums(K):
    """K = 131071 of the type's lowest value: the sum is 2^31 - 16384."""
    for m, n in ((1, 3), (18, 130), (300, 300)):
        x = torch.full((m, 131072), -128, device="cuda", dtype=torch.int8)[:, :131071]
        w = torch.full((n, 131072), -128, device="cuda", dtype=torch.int8)[:, :131071]
        one, scale = torch.ones(m, device="cuda"), torch.ones(n, device="cuda")
        got = K.gemm_i8(x, w, scale, x_scale=one, out_dtype=torch.float32)
        assert torch.all(got == float(16384 * 131071))
        w[:, ::2] = 127
        got = K.gemm_i8(x, w, scale, x_scale=one, out_dtype=torch.float32)
        assert torch.all(got == torch.tensor(-128 * (127 * 65536 - 128 * 65535), dtype=torch.float64).float().item())


def test_rows_of_a_product_that_are_not_finite(K):
    x, w, b = product(9, 20, 150, 200, torch.float32)
    x[3, 7], x[11, 0], x[19, 199] = math.nan, math.inf, -math.inf
    packed, scale = K.quantize_i8(w)
    want = quantized(x)
    got = K.gemm_i8(x, packed, scale, b)
    assert_i8(got, *want, packed, scale, b)
    assert bool(got[[3, 11, 19]].isnan().all()) and got.isnan().sum() == 3 * 150
    w[5, 1] = math.inf
    packed, scale = K.quantize_i8(w)
    assert_i8(K.gemm_i8(x, packed, scale, b), *want, packed, scale, b)


def test_scales_near_the_ends_of_fp32(K):
    """Neither order of the two scales may leave fp32 where the result does not."""
    q = torch.full((4, 64), 127, device="cuda", dtype=torch.int8)
    w = torch.full((4, 64), 100, device="cuda", dtype=torch.int8)
    big, small = torch.full((4,), 2e36, device="cuda"), torch.full((4,), 3e-37, device="cuda")
    for x_scale, scale in ((big, small), (small, big)):
        assert_i8(K.gemm_i8(q, w, scale, x_scale=x_scale, out_dtype=torch.float32), q, x_scale, w, scale)
    assert bool(K.gemm_i8(q, w, -big, x_scale=big, out_dtype=torch.float32).isneginf().all())


def test_rows_of_zeros_and_no_rows(K):
    x, w, b = product(10, 6, 40, 30, torch.bfloat16)
    packed, scale = K.quantize_i8(w)
    assert torch.equal(K.gemm_i8(torch.zeros_like(x), packed, scale, b), b.to(torch.bfloat16).expand(6, 40))
    assert K.gemm_i8(x[:0], packed, scale, b).shape == (0, 40)
    assert K.gemm_i8(x, packed[:0], scale[:0]).shape == (6, 0)
    q, s = K.quantize_i8(x[:0])
    assert q.shape == (0, 30) and s.shape == (0,) and K.gemm_i8(q, packed, scale, x_scale=s).shape == (0, 40)


def test_views_of_8_bit_rows(K):
    x, w, _ = product(11, 50, 60, 256, torch.bfloat16)
    packed, scale = K.quantize_i8(w)
    q, s = K.quantize_i8(x)
    want = K.gemm_i8(q, packed, scale, x_scale=s)
    assert torch.equal(K.gemm_i8(q[::2], packed, scale, x_scale=s[::2].contiguous()), want[::2])
    assert torch.equal(K.gemm_i8(q, packed[4:20], scale[4:20], x_scale=s), want[:, 4:20])
    assert torch.equal(K.gemm_i8(q[3:4], packed, scale, x_scale=s[3:4]), want[3:4])
    half = K.gemm_i8(q[:, 16:144], packed[:, 16:144], scale, x_scale=s, out_dtype=torch.float32)
    assert_i8(half, q[:, 16:144], s, packed[:, 16:144], scale)
    with pytest.raises(ValueError, match="16 bytes"):
        K.gemm_i8(q[:, 8:], packed[:, 8:], scale, x_scale=s)


def test_weights_and_rows_written_just_before(K):
    """The kernels start while their predecessor ends: what it writes is what they read."""
    packed = [K.quantize_i8(rows(20 + i, 2560, 4096, torch.float32, False)) for i in range(2)]
    x = [rows(30 + i, 8, 4096) for i in range(2)]
    want = [[K.gemm_i8(xi, *w) for w in packed] for xi in x]
    w, s, r = packed[0][0].clone(), packed[0][1].clone(), x[0].clone()
    for turn in range(40):
        i, j = turn & 1, turn >> 1 & 1
        w.copy_(packed[j][0])
        s.copy_(packed[j][1])
        r.copy_(x[i])
        got = K.gemm_i8(r, w, s)
        r.zero_()
        w.zero_()
        assert torch.equal(got, want[i][j])


def test_streams_and_graphs(K):
    x = [rows(40 + i, 33, 1500) for i in range(2)]
    packed, scale = K.quantize_i8(rows(42, 700, 1500, torch.float32, False))
    want = [K.gemm_i8(xi, packed, scale) for xi in x]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(K.gemm_i8(x[i], packed, scale))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])
    held = x[0].clone()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(K.gemm_i8(held, packed, scale))
        graphs.append(graph)
    for i in (1, 0, 1):
        held.copy_(x[i])
        torch.cuda.synchronize()
        for stream, graph in zip(streams, graphs):  # side by side
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want[i]) for o in outs)


def test_kernels_are_counted(K):
    from iris_b200 import _lib

    packed, scale = K.quantize_i8(rows(50, 40, 64, torch.float32))
    x = rows(51, 3, 64)
    for call, count in [(lambda: K.quantize_i8(x), 1), (lambda: K.gemm_i8(x, packed, scale), 1),
                        (lambda: K.gemm_i8(rows(52, 30, 640), *K.quantize_i8(rows(53, 40, 640))), 3),
                        (lambda: K.gemm_i8(packed[:2], packed, scale, x_scale=scale[:2]), 1),
                        (lambda: K.gemm_i8(x[:0], packed, scale), 0)]:  # fmt: skip
        before = _lib.launch_count()
        call()
        assert _lib.launch_count() - before == count


def test_error_against_the_unquantised_product(K):
    """With rows and weights rounded by at most half of a 127th of their largest magnitude."""
    x, w, _ = product(60, 64, 300, 2560, torch.bfloat16, False)
    packed, scale = K.quantize_i8(w)
    got = K.gemm_i8(x, packed, scale, out_dtype=torch.float32).double()
    a, b = x.double(), w.double()
    dx, dw = a.abs().amax(1, keepdim=True) / 254, b.abs().amax(1, keepdim=True) / 254
    most = dx * b.abs().sum(1) + (a.abs().sum(1, keepdim=True) + dx * 2560) * dw.T
    assert torch.all((got - a @ b.T).abs() <= 1.001 * most)
    assert HALF_STEP[torch.float32] < 0.001


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m, n", [(1, 75776 + 130), (32, 40000), (33, 2561), (33, 12000), (64, 15360), (65, 9473), (100, 19000), (128, 6848),
                                  (128, 40000)])  # fmt: skip
def test_short_rows_that_the_product_rounds(K, dtype, m, n):
    """Tiles of 32, 64 and 128 tokens, several of them, against rows quantised before: bit for bit."""
    packed, scale = K.quantize_i8(rows(n, n, 128, torch.float32, False))
    bias = rows(m, 1, n, torch.float32)[0]
    for k in (1, 16, 31, 48, 64, 80, 96, 128):
        x = rows(m + k, m, k, dtype)
        if m > 4:
            x[0], x[1] = 0, x[1] * torch.finfo(dtype).smallest_normal * 2.0**9
            x[2, k // 2], x[-2, 0], x[-1, -1] = math.inf, math.nan, torch.finfo(dtype).max
        q, x_scale = K.quantize_i8(x)
        for out_dtype in (dtype, torch.float32):
            want = K.gemm_i8(q, packed[:, :k], scale, bias, x_scale=x_scale, out_dtype=out_dtype)
            for view in (x, torch.cat([x[:, :1], x], dim=1)[:, 1:]):
                got = K.gemm_i8(view, packed[:, :k], scale, bias, out_dtype=out_dtype)
                assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0)) and torch.equal(got.isnan(), want.isnan())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m, k", [(10000, 300), (9600, 512), (3000, 1300), (3000, 2560), (2500, 4096), (1500, 8192), (1500, 20011)])
def test_rows_to_8_bits_in_several_turns(K, dtype, m, k):
    """More rows than teams of one, four and eight warps: the next row's values are on their way under this
    one's rounding. Rows that are not ordinary lie between the others."""
    x = rows(m, m, k, dtype)
    info = torch.finfo(dtype)
    x[5::97] = 0
    x[7::331, k // 3], x[8::331, 0], x[9::331, k - 1] = math.inf, math.nan, -math.inf
    x[10::331, k // 2], x[11::331] = info.max, info.tiny
    x[12::331] *= info.smallest_normal * 2.0**6
    assert_quantized(K, x)
    assert_quantized(K, x[:, 1:])  # rows at any value
    assert_quantized(K, x[::2])


@pytest.mark.parametrize("m", [1, 3, 40, 129, 300])
def test_a_few_tokens_by_a_vocabulary(K, m):
    """So many channels that no form gives every tile an SM's slot."""
    for n, k in [(75777, 640), (90001, 1280), (150001, 320)]:
        check(K, m, n, k, torch.bfloat16, bias=m % 2 == 1, seed=m)


def test_results_past_32_bits(K):
    m, n, k = 70001, 32768, 48
    x, w, _ = product(70, m, n, k, torch.bfloat16, False)
    packed, scale = K.quantize_i8(w)
    got = K.gemm_i8(x, packed, scale)
    assert got.numel() > 2**31
    for first in (0, 65400, m - 300):  # element 2^31 lies in row 65536
        assert torch.equal(got[first : first + 300], K.gemm_i8(x[first : first + 300], packed, scale))
    assert_i8(got[m - 300 :], *quantized(x[m - 300 :]), packed, scale)


def test_rows_and_weights_past_32_bits(K):
    gen = torch.Generator(device="cuda").manual_seed(71)
    m, k = 17000, 131071
    x = torch.randn(m, k, device="cuda", generator=gen, dtype=torch.bfloat16)
    packed, scale = K.quantize_i8(rows(72, 40, k, torch.float32, False))
    q, x_scale = K.quantize_i8(x)
    assert q.stride(0) * m > 2**31
    got = K.gemm_i8(x, packed, scale)
    assert torch.equal(got, K.gemm_i8(q, packed, scale, x_scale=x_scale, out_dtype=x.dtype))
    for first in (0, 16300, m - 100):  # byte 2^31 of q lies in row 16384
        want, want_scale = quantized(x[first : first + 100])
        assert torch.equal(q[first : first + 100].double(), want) and torch.equal(x_scale[first : first + 100], want_scale)
        assert_i8(got[first : first + 100], want, want_scale, packed, scale)
    del x, q
    n, k = 140000, 16384
    w = torch.randint(-127, 128, (n, k), device="cuda", generator=gen, dtype=torch.int8)
    scale = torch.rand(n, device="cuda", generator=gen) + 0.5
    for m in (1, 20, 300):
        x = rows(m, m, k)
        got = K.gemm_i8(x, w, scale)
        want = quantized(x)
        for first in (0, 131000, n - 100):  # byte 2^31 of w lies in row 131072
            assert_i8(got[:, first : first + 100], *want, w[first : first + 100], scale[first : first + 100])
