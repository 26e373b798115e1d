"""Builds the native parts in-tree: ``libdiffucore_b200.so``, the C-ABI library (nvcc), and
``_text_ext.so``, the torch binding of its text operators (g++ against Python's and the installed torch's
headers; left out with a message where those are missing).

The library has one translation unit per group of entry points (``csrc/dc_api.cu``: the W8A8 and
INT8 attention path, ``csrc/text_api.cu``: the text operators; each includes its kernel headers),
compiled side by side for ``sm_100a`` only and linked with the CUDA runtime statically, so the
``.so`` loads through ctypes next to PyTorch's own runtime. ``python -m diffucore_b200.build``
rebuilds what changed, ``--force`` everything.
"""

from __future__ import annotations

import os
import re
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
INCLUDE = PKG.parent / "include"
LIB = PKG / "libdiffucore_b200.so"
EXT = PKG / "_text_ext.so"
OBJECTS = PKG / "_build"

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-std=c++17", "-lineinfo",
    "-Xcompiler", "-fPIC",
]
LINK_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "--shared", "-cudart", "static"]


def _nvcc() -> str:
    home = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    cand = Path(home) / "bin" / "nvcc"
    if cand.exists():
        return str(cand)
    found = shutil.which("nvcc")
    if found is None:
        raise RuntimeError("nvcc not found: set CUDA_HOME or put nvcc on PATH")
    return found


def _sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.cuh")) + sorted(INCLUDE.glob("*.h"))


def needs_build() -> bool:
    if not LIB.exists():
        return True
    built = LIB.stat().st_mtime
    return any(p.stat().st_mtime > built for p in _sources())


def _includes(path: Path, seen: set[Path]) -> set[Path]:
    """``path`` and every file it includes by a quoted name, recursively."""
    if path not in seen and path.exists():
        seen.add(path)
        for name in re.findall(r'^#include "([^"]+)"', path.read_text(), flags=re.M):
            _includes((path.parent / name).resolve(), seen)
    return seen


def _compile(src: Path, force: bool, verbose: bool) -> Path:
    obj = OBJECTS / (src.stem + ".o")
    if not force and obj.exists():
        built = obj.stat().st_mtime
        if all(p.stat().st_mtime <= built for p in _includes(src.resolve(), set())):
            return obj
    tmp = obj.with_suffix(".o.tmp")
    _run([_nvcc(), *NVCC_FLAGS, "-c", "-o", str(tmp), str(src)], verbose)
    os.replace(tmp, obj)
    return obj


def _run(cmd: list[str], verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{Path(cmd[0]).name} failed ({res.returncode}):\n{res.stdout}\n{res.stderr}")


def build_library(force: bool = False, verbose: bool = False) -> Path:
    """Compile ``csrc/*.cu`` and link ``libdiffucore_b200.so`` unless it is up to date."""
    if not force and not needs_build():
        return LIB
    OBJECTS.mkdir(exist_ok=True)
    sources = sorted(CSRC.glob("*.cu"))
    with ThreadPoolExecutor(len(sources)) as pool:
        objects = list(pool.map(lambda src: _compile(src, force, verbose), sources))
    tmp = LIB.with_suffix(".so.tmp")
    _run([_nvcc(), *LINK_FLAGS, "-o", str(tmp), *map(str, objects)], verbose)
    os.replace(tmp, LIB)
    return LIB


def _ext_includes() -> list[Path]:
    import sysconfig

    from torch.utils import cpp_extension
    cuda = Path(os.environ.get("CUDA_HOME", "/usr/local/cuda"))
    return [*map(Path, cpp_extension.include_paths()), cuda / "include", Path(sysconfig.get_paths()["include"])]


def ext_missing() -> str | None:
    """What the binding needs beyond the library's nvcc and this machine lacks, or None."""
    if shutil.which("g++") is None:
        return "g++ not found"
    dirs = _ext_includes()
    for header in ("Python.h", "torch/extension.h", "cuda_runtime_api.h"):
        if not any((d / header).exists() for d in dirs):
            return f"{header} not found"
    return None


def _ext_stamp() -> str:
    """What a built binding is bound to besides its source: the torch and the Python it was compiled for."""
    import torch
    return f"torch {torch.__version__} abi {int(torch._C._GLIBCXX_USE_CXX11_ABI)} python {sys.version}\n"


def build_ext(force: bool = False, verbose: bool = False) -> Path:
    """Compile ``csrc/text_ext.cpp`` against the installed torch into ``_text_ext.so``, linked to the
    library beside it, unless it is up to date."""
    src = CSRC / "text_ext.cpp"
    OBJECTS.mkdir(exist_ok=True)
    stamp = OBJECTS / "text_ext.stamp"
    if not force and EXT.exists() and stamp.exists() and stamp.read_text() == _ext_stamp():
        built = EXT.stat().st_mtime
        if all(p.stat().st_mtime <= built for p in _includes(src.resolve(), set())):
            return EXT
    import torch
    lib_dir = Path(torch.__file__).resolve().parent / "lib"
    tmp = EXT.with_suffix(".so.tmp")
    _run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
          f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
          *(f"-isystem{p}" for p in _ext_includes()), str(src), "-o", str(tmp),
          f"-L{PKG}", "-l:" + LIB.name, "-Wl,-rpath,$ORIGIN", f"-L{lib_dir}", f"-Wl,-rpath,{lib_dir}",
          "-ltorch_python", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda"], verbose)
    os.replace(tmp, EXT)
    stamp.write_text(_ext_stamp())
    return EXT


def build(force: bool = False, verbose: bool = False) -> Path:
    """Everything native: the library, then the binding that links to it. Without what the binding alone
    needs, the library is built all the same and stderr says that the text operators are not."""
    lib = build_library(force, verbose)
    missing = ext_missing()
    if missing is None:
        build_ext(force, verbose)
    else:
        print(f"{EXT.name} (the text operators) not built: {missing}", file=sys.stderr)
    return lib


if __name__ == "__main__":
    force = "--force" in sys.argv
    print(build(force=force, verbose=True))
