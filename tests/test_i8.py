"""The 8-bit linear without a GPU: refusals, all before any launch."""

import ctypes
import re
import struct

import pytest
import torch

from conftest import REPO
from test_library import _einval, lib  # noqa: F401 (lib: the built library)

QUANTIZE, I8 = struct.Struct("@8q"), struct.Struct("@15q")


@pytest.fixture(scope="module")
def K(lib):  # noqa: F811
    from iris_b200 import kernels

    return kernels


def test_problem_structs_are_as_packed_here():
    text = re.sub(r"/\*.*?\*/", "", (REPO / "include" / "iris_b200.h").read_text(), flags=re.S)
    for name, packing in [("quantize", QUANTIZE), ("i8", I8)]:
        body = re.search(rf"typedef struct iris_{name}_problem {{(.*?)}}", text, flags=re.S).group(1)
        fields = sum(line.count(",") + 1 for line in filter(str.strip, body.split(";")))
        assert packing.size == 8 * fields, name


def quantize(x=16, q=16, scale=16, m=3, k=40, ldx=40, ldq=48, dtype=1):
    return "iris_quantize_i8", QUANTIZE.pack(x, q, scale, m, k, ldx, ldq, dtype), None


def product(x=16, x_scale=16, w=16, w_scale=16, bias=0, out=16, workspace=16, room=1 << 20, m=3, n=5, k=40, ldx=48, ldw=48,
            x_dtype=3, out_dtype=1):  # fmt: skip
    return I8.pack(x, x_scale, w, w_scale, bias, out, workspace, room, m, n, k, ldx, ldw, x_dtype, out_dtype)


def test_c_entries_refuse_bad_arguments(lib):  # noqa: F811
    for bad, message in [(dict(x=0), "null"), (dict(q=0), "null"), (dict(scale=0), "null"), (dict(k=0), "131071"), (dict(m=-1), "131071"),
                         (dict(k=131072, ldx=131072, ldq=131072), "131071"), (dict(ldx=-1), "stride"), (dict(ldq=44), "multiples"),
                         (dict(ldq=32), "multiples"), (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(q=20), "misaligned"),
                         (dict(x=17), "misaligned"), (dict(x=18, dtype=0), "misaligned"), (dict(scale=18), "misaligned")]:  # fmt: skip
        assert message in _einval(lib, *quantize(**bad)), bad
    assert "null" in _einval(lib, "iris_quantize_i8", None, None)
    assert lib.iris_quantize_i8(quantize(m=0, x=0)[1], None) == 0

    for bad, message in [(dict(x=0), "null"), (dict(x_scale=0), "null"), (dict(w=0), "null"), (dict(w_scale=0), "null"),
                         (dict(out=0), "null"), (dict(k=0), "131071"), (dict(k=131072, ldx=131072, ldw=131072), "int32"),
                         (dict(m=-1), "sizes"), (dict(n=-1), "sizes"), (dict(ldw=44), "16 bytes"), (dict(ldw=32), "16 bytes"),
                         (dict(w=24), "16 bytes"), (dict(x=24), "16 bytes"), (dict(ldx=56), "16 bytes"), (dict(ldx=32), "16 bytes"),
                         (dict(x_dtype=4), "dtype"), (dict(out_dtype=3), "dtype"), (dict(w_scale=18), "misaligned"),
                         (dict(bias=18), "misaligned"), (dict(out=17), "misaligned"), (dict(out=18, out_dtype=0), "misaligned"),
                         (dict(x_dtype=1, m=300, workspace=0), "workspace"), (dict(x_dtype=1, m=300, workspace=24), "workspace"),
                         (dict(x_dtype=1, m=300, room=15599), "workspace"), (dict(x_dtype=1, ldx=-1), "stride"),
                         (dict(x_dtype=0, x=18), "misaligned")]:  # fmt: skip
        assert message in _einval(lib, "iris_gemm_i8", product(**bad), None), bad
    for name in ("iris_gemm_i8", "iris_gemm_i8_workspace"):
        assert "null" in _einval(lib, name, None, None)
    for empty in (dict(m=0), dict(n=0)):
        assert lib.iris_gemm_i8(product(x=0, **empty), None) == 0


def test_workspace_is_for_rows_that_are_quantised(lib):  # noqa: F811
    def need(**sizes):
        out = ctypes.c_int64(-1)
        assert lib.iris_gemm_i8_workspace(product(**sizes), ctypes.byref(out)) == 0
        return out.value

    assert need() == 0
    for dtype in (0, 1, 2):  # rows at 16 bytes, then their scales
        assert need(x_dtype=dtype, m=300) == 300 * 48 + 1200
        assert need(x_dtype=dtype, m=1000, k=16) == 16000 + 4000
        assert need(x_dtype=dtype, k=7000, ldx=7008, ldw=7008) == 3 * 7008 + 16
        # a few rows are rounded by the product itself
        for m in (3, 30, 100, 128):
            assert need(x_dtype=dtype, m=m) == 0
        assert need(x_dtype=dtype, m=0) == need(x_dtype=dtype, n=0, m=1000) == 0


def test_wrappers_refuse_before_any_launch(K):
    x, w = torch.zeros(3, 32), torch.zeros(5, 32, dtype=torch.int8)
    scale, rows = torch.zeros(5), torch.zeros(3)
    with pytest.raises(ValueError, match="CUDA"):
        K.quantize_i8(x)
    for bad, message in [(x[0], "M, K"), (x.double(), "dtype"), (w, "dtype"), (x[:, ::2], "contiguous"), (3, "M, K")]:
        with pytest.raises(ValueError, match=message):
            K.quantize_i8(bad)
    with pytest.raises(ValueError, match="CUDA"):
        K.gemm_i8(x, w, scale)
    eight = w[:3]
    for args, kw, message in [
        ((x[0], w, scale), {}, "M, K"),
        ((x, w[0], scale), {}, "M, K"),
        ((x, w.float(), scale), {}, "packed must be int8"),
        ((x, w[:, :16], scale), {}, "packed must be int8"),
        ((x[:, ::2], w[:, :16], scale), {}, "rows must be contiguous"),
        ((x[:, :16], w[:, ::2], scale), {}, "rows must be contiguous"),
        ((x, w, scale[:4]), {}, "scale must be"),
        ((x, w, scale.half()), {}, "scale must be"),
        ((x, w, scale[:, None]), {}, "scale must be"),
        ((x, w, scale, rows), {}, "bias must be"),
        ((x, w, scale, scale.double()), {}, "bias must be"),
        ((x, w, scale), {"x_scale": rows}, "x_scale goes with"),
        ((eight, w, scale), {}, "x_scale goes with"),
        ((eight, w, scale), {"x_scale": scale}, "x_scale must be"),
        ((eight, w, scale), {"x_scale": rows.half()}, "x_scale must be"),
        ((x.double(), w, scale), {}, "dtype"),
        ((x, w, scale), {"out_dtype": torch.int8}, "dtype"),
        ((x, w, scale), {"out_dtype": 3}, "dtype"),
        ((x, w, None), {}, "needs x"),
    ]:
        with pytest.raises(ValueError, match=message):
            K.gemm_i8(*args, **kw)


def test_which_rows_the_product_rounds(lib):  # noqa: F811
    """Calls of one launch need no workspace; where the device is done earlier with two, there are two."""

    def rounds(m, n, k, dtype):
        out, ld = ctypes.c_int64(-1), (k + 15) // 16 * 16
        assert lib.iris_gemm_i8_workspace(product(m=m, n=n, k=k, ldx=k, ldw=ld, x_dtype=dtype), ctypes.byref(out)) == 0
        assert out.value in (0, m * ld + (m + 3) // 4 * 16)
        return out.value == 0

    for dtype in (1, 2):  # 16 bits
        for m, n, k in [(1, 2560, 2560), (4, 2560, 2560), (8, 2560, 1280), (1, 256, 10240), (3, 40000, 1280), (1, 40000, 16), (32, 150000, 128),
                        (128, 2560, 128), (64, 15360, 128), (64, 70000, 80), (128, 15360, 80), (128, 70000, 40)]:  # fmt: skip
            assert rounds(m, n, k, dtype), (m, n, k)
        for m, n, k in [(16, 2560, 640), (8, 2560, 640), (5, 2560, 300), (64, 2560, 160), (17, 256, 600), (4, 40000, 640),
                        (1, 150000, 1280), (128, 15360, 128), (64, 40000, 128), (128, 40000, 64), (129, 5, 16), (2, 2560, 20000)]:  # fmt: skip
            assert not rounds(m, n, k, dtype), (m, n, k)
    for m, n, k in [(1, 2560, 4096), (4, 6848, 1280), (32, 2560, 64), (1, 256, 10240)]:  # fp32
        assert rounds(m, n, k, 0), (m, n, k)
    for m, n, k in [(4, 2560, 640), (4, 256, 2560), (3, 2560, 3000), (17, 256, 128), (128, 15360, 64)]:
        assert not rounds(m, n, k, 0), (m, n, k)
