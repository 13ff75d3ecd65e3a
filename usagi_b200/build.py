"""Ahead-of-time build of the sm_100a kernel library (``libbsattn.so``, in-tree).

The reference JIT-compiled Triton variants at first call and precompiled stride classes in
``setup()`` (kernels/v4_leaderboard_0740ms.py:189-238).  Here the CUDA source is compiled once,
for sm_100a only, with nvcc; the CUDA runtime is linked statically and the driver entry point
for TMA descriptors is resolved at run time, so the library loads on hosts without a GPU.

Usage: ``python -m usagi_b200.build [--force]``
"""
from __future__ import annotations

import hashlib
import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
CSRC = PKG_DIR / "csrc"
INCLUDE = PKG_DIR.parent / "include"
LIB_NAME = "libbsattn.so"
LIB_PATH = PKG_DIR / LIB_NAME
# Hash of the sources, headers and flags the in-tree library was built from (written next to it).
STAMP_PATH = PKG_DIR / (LIB_NAME + ".sha256")

SOURCES = ["bsattn_fwd.cu", "csr_build.cu", "peer.cu", "paged_append.cu", "paged_attn.cu",
           "paged_few.cu", "paged_tile.cu"]
HEADERS = ["sm100_ptx.cuh", "paged_common.cuh", "paged_few.cuh", "paged_tile.cuh"]

# The Python side of the paged-cache calls: a CPython module of its own, compiled against torch, which
# reaches the kernel library through the addresses that _lib gives it.
BINDING_NAME = "_paged_binding.so"
BINDING_PATH = PKG_DIR / BINDING_NAME
BINDING_STAMP_PATH = PKG_DIR / (BINDING_NAME + ".sha256")
BINDING_SOURCE = CSRC / "paged_binding.cpp"
BINDING_FLAGS = ["-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden"]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo",
    "-O3",
    "-std=c++17",
    "-Xcompiler", "-fPIC",
    "-Xcompiler", "-fvisibility=hidden",
    "-cudart", "static",
    "-shared",
]


def _nvcc() -> str:
    cand = [os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"]
    for c in cand:
        if c and os.path.exists(c):
            return c
    raise RuntimeError("nvcc not found: the sm_100a kernel library cannot be built")


def _inputs():
    files = [CSRC / s for s in SOURCES] + [CSRC / h for h in HEADERS] + [INCLUDE / "bsattn.h"]
    return files


def source_hash() -> str:
    """sha256 over the compile flags and the bytes of every source and header of the library."""
    h = hashlib.sha256()
    h.update(" ".join(NVCC_FLAGS).encode())
    for f in _inputs():
        h.update(f.name.encode())
        h.update(f.read_bytes())
    return h.hexdigest()


def needs_build() -> bool:
    """True unless the in-tree library exists and its stamp names the current sources: a library
    built from other sources (whatever its file time) is rebuilt."""
    if not LIB_PATH.exists() or not STAMP_PATH.exists():
        return True
    return STAMP_PATH.read_text().strip() != source_hash()


def binding_hash() -> str:
    """sha256 over what the binding is built from: flags, sources, torch's and Python's versions."""
    import torch
    h = hashlib.sha256()
    h.update(" ".join([*BINDING_FLAGS, torch.__version__, sys.version]).encode())
    for f in (BINDING_SOURCE, INCLUDE / "bsattn.h"):
        h.update(f.read_bytes())
    return h.hexdigest()


def binding_needs_build() -> bool:
    """As :func:`needs_build`, for the binding."""
    if not BINDING_PATH.exists() or not BINDING_STAMP_PATH.exists():
        return True
    return BINDING_STAMP_PATH.read_text().strip() != binding_hash()


def _run(cmd, verbose: bool) -> str:
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed ({res.returncode}):\n{res.stdout}\n{res.stderr}")
    return res.stderr


def build_binding(force: bool = False, verbose: bool = False) -> Path:
    """Compile ``csrc/paged_binding.cpp`` into ``usagi_b200/_paged_binding.so``; returns its path."""
    if not force and not binding_needs_build():
        return BINDING_PATH
    import sysconfig

    import torch
    root = Path(torch.__file__).parent
    nvcc = Path(_nvcc()).resolve()
    tmp = BINDING_PATH.with_suffix(".so.tmp")
    _run([os.environ.get("CXX") or "g++", *BINDING_FLAGS,
          f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
          "-isystem", sysconfig.get_paths()["include"], "-isystem", str(root / "include"),
          "-isystem", str(nvcc.parent.parent / "include"), str(BINDING_SOURCE), "-o", str(tmp),
          "-L", str(root / "lib"), "-ltorch_python", "-ltorch_cpu", "-ltorch", "-lc10", "-lc10_cuda"],
         verbose)
    digest = binding_hash()
    os.replace(tmp, BINDING_PATH)
    BINDING_STAMP_PATH.write_text(digest + "\n")
    return BINDING_PATH


def build(force: bool = False, verbose: bool = False, ptxas_info: bool = False) -> Path:
    """Compile ``csrc/*.cu`` into ``usagi_b200/libbsattn.so`` and the binding next to it; returns the
    library path.  The library needs only nvcc; where the binding cannot be built (no headers of Python
    or torch) that is printed, and the paged-cache calls of Python are missing."""
    _build_library(force, verbose, ptxas_info)
    try:
        build_binding(force, verbose)
    except (ImportError, OSError, RuntimeError) as e:
        BINDING_PATH.unlink(missing_ok=True)  # one of other sources must not meet this library
        print(f"usagi_b200: no paged-cache calls, their binding was not built: {e}", file=sys.stderr)
    return LIB_PATH


def _build_library(force: bool, verbose: bool, ptxas_info: bool) -> None:
    if not force and not needs_build():
        return
    cmd = [_nvcc(), *NVCC_FLAGS]
    if ptxas_info:
        cmd += ["-Xptxas", "-v"]
    tmp = LIB_PATH.with_suffix(".so.tmp")
    cmd += ["-o", str(tmp)] + [str(CSRC / s) for s in SOURCES]
    stderr = _run(cmd, verbose)
    if verbose or ptxas_info:
        sys.stdout.write(stderr)
    digest = source_hash()
    os.replace(tmp, LIB_PATH)
    STAMP_PATH.write_text(digest + "\n")


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True, ptxas_info="--ptxas" in sys.argv)
    print(LIB_PATH)
