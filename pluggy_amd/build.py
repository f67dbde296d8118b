"""Build ``pluggy_amd/libpmoe.so`` from ``pluggy_amd/csrc/*.hip`` with hipcc (gfx950), and
``pluggy_amd/_autograd.so``, the C++ autograd nodes over it, from ``csrc/autograd.cpp``.

Usage: ``python -m pluggy_amd.build`` (or ``__graft_entry__.build()``). Each
translation unit compiles in parallel into ``pluggy_amd/_build/``; the shared
libraries are then linked in place, next to the package, so they travel with the
source tree. The nodes are built for the torch that is importable.
"""

from __future__ import annotations

import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
BUILD = PKG / "_build"
LIB = PKG / "libpmoe.so"
NODES = PKG / "_autograd.so"
ARCH = os.environ.get("PMOE_OFFLOAD_ARCH", "gfx950")

HIPCC_FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-fvisibility=hidden",
    # packed fp32 ops are kept out of every kernel (they have given wrong
    # results on this hardware pool); the host pass warns that it does not know
    # the feature, which is harmless.
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall",
    "-Wno-unused-function",
]


def hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("hipcc not found: the pmoe HIP library cannot be built")


def _compile(src: Path) -> Path:
    obj = BUILD / (src.stem + ".o")
    cmd = [hipcc(), *HIPCC_FLAGS, "-c", str(src), "-o", str(obj)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    noise = "is not a recognized feature for this target"
    err = "\n".join(l for l in res.stderr.splitlines() if noise not in l)
    if res.returncode != 0:
        raise RuntimeError(f"hipcc failed on {src.name}:\n{err}")
    if err.strip():
        print(err, file=sys.stderr)
    return obj


def _run(cmd: list[str], what: str) -> None:
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{what} failed:\n{res.stderr}")


def _cxx() -> str:
    return os.environ.get("CXX", "g++")


def _compile_nodes() -> Path:
    import torch
    from torch.utils import cpp_extension

    obj = BUILD / "autograd.o"
    includes = (*cpp_extension.include_paths(), sysconfig.get_paths()["include"])
    _run([_cxx(), "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-Wall", "-DTORCH_EXTENSION_NAME=_autograd",
          f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *(f"-isystem{p}" for p in includes),
          "-c", str(CSRC / "autograd.cpp"), "-o", str(obj)], "the compilation of autograd.cpp")
    return obj


def _link_nodes(obj: Path) -> None:
    from torch.utils import cpp_extension

    tmp = NODES.with_suffix(".so.tmp")
    libs = cpp_extension.library_paths()
    _run([_cxx(), "-shared", str(obj), "-o", str(tmp), f"-L{PKG}", "-l:libpmoe.so", *(f"-L{p}" for p in libs),
          "-ltorch", "-ltorch_cpu", "-lc10", "-ltorch_python", "-Wl,-rpath,$ORIGIN", *(f"-Wl,-rpath,{p}" for p in libs)],
         "the link of _autograd.so")
    os.replace(tmp, NODES)


def build(verbose: bool = True) -> Path:
    BUILD.mkdir(exist_ok=True)
    sources = sorted(CSRC.glob("*.hip"))
    if not sources:
        raise RuntimeError(f"no HIP sources under {CSRC}")
    with cf.ThreadPoolExecutor(max_workers=min(8, len(sources) + 1)) as ex:
        nodes = ex.submit(_compile_nodes)
        objs = list(ex.map(_compile, sources))
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", *map(str, objs), "-o", str(tmp)]
    _run(cmd, "link")
    os.replace(tmp, LIB)
    _link_nodes(nodes.result())
    if verbose:
        print(f"built {LIB} ({LIB.stat().st_size / 1e6:.1f} MB) from {len(sources)} sources for {ARCH}")
    return LIB


if __name__ == "__main__":
    build()
