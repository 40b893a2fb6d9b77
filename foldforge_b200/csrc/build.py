"""Build ``foldforge_b200/_ffb.so`` from the CUDA sources with nvcc for sm_100a only.

``python -m foldforge_b200.csrc.build`` (or ``__graft_entry__.build()``). The library is
built in-tree so it travels with the repository snapshot; nvcc cross-compiles without a
GPU. Each translation unit is compiled to an object in ``_build/`` and relinked only when
a source or header changed.
"""

from __future__ import annotations

import os
import subprocess
import sys
from pathlib import Path

HERE = Path(__file__).resolve().parent
PKG = HERE.parent
OUT = PKG / "_ffb.so"
BINDING = PKG / "_binding.so"
BUILD = PKG.parent / "_build"
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr", "-Xptxas", "-v"]


def sources() -> list[Path]:
    return sorted(HERE.glob("*.cu"))


def _newest_header() -> float:
    hs = list(HERE.glob("*.h")) + list(HERE.glob("*.cuh")) + list((PKG.parent / "include").glob("*.h"))
    return max((h.stat().st_mtime for h in hs), default=0.0)


def build(verbose: bool = False) -> Path:
    nvcc = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
    BUILD.mkdir(exist_ok=True)
    objs = []
    header_time = _newest_header()
    for src in sources():
        obj = BUILD / (src.stem + ".o")
        objs.append(obj)
        if obj.exists() and obj.stat().st_mtime >= max(src.stat().st_mtime, header_time):
            continue
        cmd = [nvcc, *ARCH, *FLAGS, "-c", str(src), "-o", str(obj)]
        res = subprocess.run(cmd, capture_output=True, text=True)
        log = BUILD / (src.stem + ".ptxas.txt")
        log.write_text(res.stdout + res.stderr)
        if res.returncode != 0:
            sys.stderr.write(res.stdout + res.stderr)
            raise RuntimeError(f"nvcc failed on {src.name}")
        if verbose:
            sys.stderr.write(res.stderr)
    if not OUT.exists() or OUT.stat().st_mtime < max(o.stat().st_mtime for o in objs):
        cmd = [nvcc, *ARCH, "-shared", "-Xcompiler", "-fPIC", "-o", str(OUT), *map(str, objs)]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            sys.stderr.write(res.stdout + res.stderr)
            raise RuntimeError("nvcc link failed")
    build_binding()
    return OUT


def build_binding() -> Path:
    """``foldforge_b200/_binding.so``: the torch-facing calls of ``binding.cpp``, against the installed torch."""
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    src, header = HERE / "binding.cpp", PKG.parent / "include" / "foldforge_b200.h"
    newest = max(src.stat().st_mtime, header.stat().st_mtime, Path(torch.__file__).stat().st_mtime)
    if BINDING.exists() and BINDING.stat().st_mtime >= newest:
        return BINDING
    includes = [*cpp_extension.include_paths(), "/usr/local/cuda/include", sysconfig.get_paths()["include"]]
    libs = Path(torch.__file__).parent / "lib"
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-DTORCH_API_INCLUDE_EXTENSION_H",
           *[f"-I{p}" for p in includes], str(src), "-o", str(BINDING), f"-L{libs}", f"-Wl,-rpath,{libs}", "-lc10", "-lc10_cuda",
           "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python", "-ltorch"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("the compiler failed on binding.cpp")
    return BINDING


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
