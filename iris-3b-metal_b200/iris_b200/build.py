"""Build ``libiris_b200.so`` in-tree with nvcc for sm_100a.

    python -m iris_b200.build            # from the iris-3b-metal_b200 directory

The library is one translation unit (``csrc/iris_b200.cu``); the output lands
next to this file so it travels with the source tree. So does ``_text_side.*.so``
(``csrc/text_side.cpp``), the CPython module through which the text side's per-token
calls reach the library, built by the host compiler against torch's headers; its name
holds the Python and torch that it is for.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
import warnings
from pathlib import Path

from iris_b200 import _lib

PACKAGE = Path(__file__).resolve().parent
CSRC = PACKAGE.parent / "csrc"
INCLUDE = PACKAGE.parent.parent / "include"
LIBRARY = PACKAGE / "libiris_b200.so"
MODULE = _lib.TEXT_SIDE
MODULE_SOURCE = CSRC / "text_side.cpp"

NVCC_FLAGS = [
    "-gencode",
    "arch=compute_100a,code=sm_100a",
    "-lineinfo",
    "-O3",
    "-std=c++17",
    "-Xcompiler",
    "-fPIC",
    "-shared",
]


def nvcc() -> str:
    found = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(found).exists():
        raise RuntimeError("nvcc not found; the CUDA toolkit is needed to build libiris_b200.so")
    return found


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h")) + [INCLUDE / "iris_b200.h"]


def up_to_date() -> bool:
    if not LIBRARY.exists():
        return False
    built = LIBRARY.stat().st_mtime
    return all(src.stat().st_mtime <= built for src in sources())


def module_up_to_date() -> bool:
    if not MODULE.exists():
        return False
    built = MODULE.stat().st_mtime
    return all(src.stat().st_mtime <= built for src in (MODULE_SOURCE, INCLUDE / "iris_b200.h"))


def _run(cmd: list[str], target: Path, verbose: bool) -> None:
    """Run a compiler that writes ``target`` (renamed into place when it is whole)."""
    tmp = target.with_suffix(f".so.tmp{os.getpid()}")
    result = subprocess.run([*cmd, "-o", str(tmp)], capture_output=True, text=True)
    if result.returncode != 0:
        raise RuntimeError(f"{Path(cmd[0]).name} failed ({result.returncode}):\n{result.stderr[-4000:]}")
    if verbose:
        sys.stderr.write(result.stderr)
    os.replace(tmp, target)


def build_module(force: bool = False, verbose: bool = False) -> Path:
    if not force and module_up_to_date():
        return MODULE
    import torch

    root = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc()).resolve().parents[1]
    includes = [root / "include", root / "include/torch/csrc/api/include", cuda / "include", sysconfig.get_paths()["include"]]
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *(f"-isystem{i}" for i in includes),
           str(MODULE_SOURCE), f"-L{root / 'lib'}", "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"]  # fmt: skip
    try:
        _run(cmd, MODULE, verbose)
    except (RuntimeError, OSError):
        MODULE.unlink(missing_ok=True)  # none of an older source is left
        raise
    return MODULE


def build(force: bool = False, verbose: bool = False) -> Path:
    """The library, then the module. The engine needs the library alone, so that a
    host without Python's or torch's headers still builds it: it is warned, and the text
    side's calls raise there."""
    if force or not up_to_date():
        cmd = [nvcc(), *NVCC_FLAGS, f"-I{INCLUDE}", str(CSRC / "iris_b200.cu")]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
        _run(cmd, LIBRARY, verbose)
    try:
        build_module(force, verbose)
    except (RuntimeError, OSError) as e:
        warnings.warn(f"{MODULE.name} is not built, the text side's calls will raise: {e}", stacklevel=2)
    return LIBRARY


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
