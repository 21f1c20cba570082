"""Builds libfpx.so (the C-ABI library) in-tree with nvcc for sm_100a, and _paged.so, the
paged cache's binding to torch tensors, with the host compiler.

    python -m exp3_b200.build [--force]

Each ``csrc/*.cu`` compiles in parallel to an object under ``_build/``; the shared
library links them with the static CUDA runtime. A rebuild happens only when a
source or header is newer than what it builds.
"""

from __future__ import annotations

import concurrent.futures
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
BUILD = ROOT / "_build"
LIB = PKG / "libfpx.so"
BINDING_SOURCE = PKG / "binding" / "paged.cpp"
BINDING = PKG / "_paged.so"
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
         "-I", str(ROOT / "include")]


def nvcc() -> str:
    found = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(found).exists():
        raise RuntimeError("nvcc not found; the CUDA toolkit is needed to build libfpx")
    return found


def sources():
    return sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.cpp"))


def _stale() -> bool:
    if not LIB.exists():
        return True
    newest = max(p.stat().st_mtime for p in list(CSRC.iterdir()) + list((ROOT / "include").iterdir()))
    return newest > LIB.stat().st_mtime


def _compile(src: Path) -> Path:
    obj = BUILD / (src.stem + ".o")
    cmd = [nvcc(), *ARCH, *FLAGS, "-c", str(src), "-o", str(obj)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src.name}:\n{res.stderr}")
    return obj


def _binding_stale() -> bool:
    if not BINDING.exists():
        return True
    return max(p.stat().st_mtime for p in (BINDING_SOURCE, ROOT / "include" / "fpx.h")) > BINDING.stat().st_mtime


def _build_binding() -> None:
    import torch

    root = Path(torch.__file__).parent
    cuda = Path(nvcc()).resolve().parents[1]
    tmp = BINDING.with_suffix(".so.tmp")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I", str(ROOT / "include"),
           "-isystem", str(root / "include"), "-isystem", str(root / "include" / "torch" / "csrc" / "api" / "include"),
           "-isystem", sysconfig.get_paths()["include"], "-isystem", str(cuda / "include"), str(BINDING_SOURCE),
           "-o", str(tmp), "-L", str(root / "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed on {BINDING_SOURCE.name}:\n{res.stderr}")
    tmp.replace(BINDING)


def _build_library() -> None:
    BUILD.mkdir(exist_ok=True)
    with concurrent.futures.ThreadPoolExecutor(max_workers=os.cpu_count() or 4) as pool:
        objs = list(pool.map(_compile, sources()))
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [nvcc(), *ARCH, "-shared", "-o", str(tmp), *map(str, objs)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stderr}")
    tmp.replace(LIB)


def build(force: bool = False, verbose: bool = False) -> Path:
    todo = [step for step, stale in ((_build_library, _stale()), (_build_binding, _binding_stale())) if force or stale]
    with concurrent.futures.ThreadPoolExecutor(max_workers=2) as pool:
        list(pool.map(lambda step: step(), todo))
    if todo and verbose:
        print(f"built {LIB}, {BINDING.name}")
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True)
