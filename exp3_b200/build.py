"""Builds libfpx.so (the C-ABI library) in-tree with nvcc for sm_100a, and _paged.so, the
paged cache's binding to torch tensors, with the host compiler.

    python -m exp3_b200.build [--force] [--library]

Each ``csrc/*.cu`` compiles in parallel to an object under ``_build/``; the shared
library links them with the static CUDA runtime. A rebuild happens only when a
source or header is newer than what it builds, and of the binding also when it was built for
another torch or Python. ``--library`` builds the library alone, which needs nvcc only; so does a
build where torch is not installed.
"""

from __future__ import annotations

import concurrent.futures
import importlib.metadata
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


def _binding_for() -> str | None:
    """What the binding is built for (it links torch's own C++ functions); None: torch is not installed."""
    try:
        return f"torch {importlib.metadata.version('torch')} {sys.implementation.cache_tag}"
    except importlib.metadata.PackageNotFoundError:
        return None


def _binding_stale() -> bool:
    built_for = BUILD / "paged_binding.txt"
    if not BINDING.exists() or not built_for.exists() or built_for.read_text() != _binding_for():
        return True
    return max(p.stat().st_mtime for p in (BINDING_SOURCE, ROOT / "include" / "fpx.h")) > BINDING.stat().st_mtime


def _build_binding() -> None:
    import torch

    root = Path(torch.__file__).parent
    cuda = Path(nvcc()).resolve().parents[1]
    tmp = BINDING.with_suffix(".so.tmp")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f'-DFPX_TORCH_VERSION="{torch.__version__}"',
           "-I", str(ROOT / "include"),
           "-isystem", str(root / "include"), "-isystem", str(root / "include" / "torch" / "csrc" / "api" / "include"),
           "-isystem", sysconfig.get_paths()["include"], "-isystem", str(cuda / "include"), str(BINDING_SOURCE),
           "-o", str(tmp), "-L", str(root / "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed on {BINDING_SOURCE.name}:\n{res.stderr}")
    tmp.replace(BINDING)
    BUILD.mkdir(exist_ok=True)
    (BUILD / "paged_binding.txt").write_text(_binding_for() or "")


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


def build(force: bool = False, verbose: bool = False, library_only: bool = False) -> Path:
    """The library, and the binding unless ``library_only`` or torch is not installed. A binding that does not build leaves the
    library built, for users of the C ABI, and raises."""
    binding = not library_only and _binding_for() is not None
    todo = [(_build_library, LIB)] if force or _stale() else []
    if binding and (force or _binding_stale()):
        todo.append((_build_binding, BINDING))
    with concurrent.futures.ThreadPoolExecutor(max_workers=2) as pool:
        steps = [pool.submit(step) for step, _ in todo]
    for step, (_, path) in zip(steps, todo):  # the library's first
        step.result()
        if verbose:
            print(f"built {path}")
    if verbose and not binding and not library_only:
        print(f"torch is not installed: {BINDING.name} is not built")
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True, library_only="--library" in sys.argv)
