"""Attention behind a shared prefix without a GPU: refusals, all before any launch."""

import ctypes
import math
import re
import struct

import pytest
import torch

from conftest import REPO
from test_library import _einval, lib  # noqa: F401 (lib: the built library)

PREFIX = struct.Struct("@38qd")


@pytest.fixture(scope="module")
def K(lib):  # noqa: F811
    from iris_b200 import kernels

    return kernels


def test_problem_struct_is_as_packed_here():
    text = re.sub(r"/\*.*?\*/", "", (REPO / "include" / "iris_b200.h").read_text(), flags=re.S)
    body = re.search(r"typedef struct iris_prefix_problem {(.*?)}", text, flags=re.S).group(1)
    fields = sum((line.count(",") + 1) * (4 if "iris_head_rows" in line else 1) for line in filter(str.strip, body.split(";")))
    assert PREFIX.size == 8 * fields


def attend(q=16, dtype=1, batch=6, groups=2, heads=4, kv=2, n=3, p=7, m=5, dim=128, qn=128, pn=128, kn=128, vb=0, right=0,
           scale=0.1, out=16, on=512, workspace=0, room=0):  # fmt: skip
    def rows(data=16, b=0, h=0, n=128):
        return data, b, h, n

    return PREFIX.pack(*rows(q, n=qn), *rows(n=pn), *rows(), *rows(n=kn), *rows(b=vb), out, 0, on, 0, 0, 0, workspace, room, dtype,
                       batch, groups, heads, kv, n, p, m, dim, right, scale)  # fmt: skip


def test_c_entries_refuse_bad_arguments(lib):  # noqa: F811
    for bad, message in [(dict(dtype=0), "bf16 or f16"), (dict(heads=3), "multiple of heads_kv"), (dict(dim=80), "head_dim"),
                         (dict(qn=12), "16 bytes"), (dict(q=8), "16 bytes"), (dict(pn=12), "16 bytes"), (dict(on=12), "16 bytes"),
                         (dict(out=24), "16 bytes"), (dict(right=-2), "right"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
                         (dict(scale=math.nan), "scale"), (dict(scale=math.inf), "scale"), (dict(scale=3e38), "scale"),
                         (dict(m=1 << 30), "sizes"), (dict(p=1 << 30), "sizes"), (dict(n=1 << 30), "sizes"), (dict(p=-1), "sizes"),
                         (dict(batch=65536), "sizes"), (dict(groups=0), "groups"), (dict(groups=4), "groups"), (dict(kv=0), "heads_kv"),
                         (dict(qn=0), "repeat"), (dict(pn=0), "repeat"), (dict(kn=0), "repeat"), (dict(vb=-128), "repeat"),
                         (dict(kn=1 << 34), "apart"), (dict(q=0), "null"), (dict(out=0), "null")]:  # fmt: skip
        assert message in _einval(lib, "iris_prefix_attn_fwd", attend(**bad), None), bad
    for name in ("iris_prefix_attn_fwd", "iris_prefix_attn_workspace"):
        assert "null" in _einval(lib, name, None, None)
    for empty in (dict(batch=0), dict(n=0)):
        assert lib.iris_prefix_attn_fwd(attend(q=0, out=0, **empty), None) == 0


def test_workspace_is_refused_for_bad_sizes_too(lib):  # noqa: F811
    out = ctypes.c_int64(-1)
    assert lib.iris_prefix_attn_workspace(attend(), ctypes.byref(out)) == 0 and out.value >= 0
    for bad in (dict(groups=5), dict(dim=96), dict(heads=3)):
        assert lib.iris_prefix_attn_workspace(attend(**bad), ctypes.byref(out)) == 1


def test_wrapper_refuses_before_any_launch(K):
    def t(*shape):
        return torch.zeros(*shape, dtype=torch.bfloat16)

    def int32(n):
        return torch.zeros(n, dtype=torch.int32)

    good = dict(q=t(6, 4, 3, 64), prefix_k=t(2, 2, 7, 64), prefix_v=t(2, 2, 7, 64), k=t(6, 2, 5, 64), v=t(6, 2, 5, 64))
    with pytest.raises(ValueError, match="CUDA"):
        K.prefix_attention(**good)
    for bad, message in [
        (dict(q=t(4, 3, 64)), "q .B, H, N, D"),
        (dict(q=t(6, 4, 3, 64).float()), "bf16, f16"),
        (dict(v=t(6, 2, 5, 64).half()), "bf16, f16"),
        (dict(prefix_v=t(2, 2, 7, 64).half()), "bf16, f16"),
        (dict(q=t(6, 4, 3, 32)), "head_dim"),
        (dict(q=t(5, 4, 3, 64)), "multiple of the prefixes"),
        (dict(prefix_k=t(0, 2, 7, 64)), "multiple of the prefixes"),
        (dict(prefix_k=t(4, 2, 7, 64)), "multiple of the prefixes"),
        (dict(prefix_v=t(2, 2, 8, 64)), "prefix_v must be"),
        (dict(prefix_v=t(1, 2, 7, 64)), "prefix_v must be"),
        (dict(k=t(5, 2, 5, 64)), "k must be"),
        (dict(k=t(6, 1, 5, 64)), "k must be"),
        (dict(v=t(6, 2, 6, 64)), "v must be"),
        (dict(k=t(6, 2, 5, 128)[..., ::2]), "contiguous"),
        (dict(prefix_lengths=int32(3)), "prefix_lengths must be"),
        (dict(prefix_lengths=int32(2).long()), "prefix_lengths must be"),
        (dict(starts=int32(2)), "starts must be"),
        (dict(lengths=int32(12)[::2]), "lengths must be"),
        (dict(right=-1), "right must not be"),
        (dict(out=good["q"]), "q's own rows"),
    ]:
        with pytest.raises(ValueError, match=message):
            K.prefix_attention(**{**good, **bad})
    for name in ("prefix_k", "prefix_v", "k", "v"):
        with pytest.raises(ValueError, match="keys or values"):
            K.prefix_attention(**good, out=good[name].view(-1)[: 6 * 64].view(6, 1, 64))
    with pytest.raises(TypeError):
        K.prefix_attention(**good, scale="x")


def test_strides_of_lone_entries_are_not_looked_at(lib):  # noqa: F811
    """Up to the check that refuses a missing output, which comes after those of the strides."""
    for stride in (1 << 34, -(1 << 40), 12, -128):
        assert "null" in _einval(lib, "iris_prefix_attn_fwd", attend(m=1, kn=stride, out=0), None), stride
        assert "null" in _einval(lib, "iris_prefix_attn_fwd", attend(p=1, pn=stride, out=0), None), stride
        assert "null" in _einval(lib, "iris_prefix_attn_fwd", attend(n=1, qn=stride, out=0), None), stride
        assert "null" in _einval(lib, "iris_prefix_attn_fwd", attend(batch=1, groups=1, vb=stride, out=0), None), stride


def test_keys_that_32_bits_do_not_count_are_refused(lib):  # noqa: F811
    """A row tile's place among all keys, and one chunk of them, are held in 32 bits."""
    out = ctypes.c_int64(-1)
    for p, m in [(1 << 29, 1 << 29), ((1 << 30) - 1, 1), ((1 << 30) - 1, (1 << 30) - 1), (5, (1 << 30) - 5)]:
        assert "sizes" in _einval(lib, "iris_prefix_attn_fwd", attend(p=p, m=m), None)
        assert "sizes" in _einval(lib, "iris_prefix_attn_workspace", attend(p=p, m=m), ctypes.byref(out))
    assert lib.iris_prefix_attn_workspace(attend(p=1 << 29, m=(1 << 29) - 1), ctypes.byref(out)) == 0
