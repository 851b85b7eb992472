"""Builds the sm_100a shared library `libdory_decode.so` next to this file.

The library is plain C ABI (include/dory_decode.h) linked against the CUDA runtime only;
the Python host code loads it with ctypes, so no torch headers are involved and the same
.so serves a C, C++ or Python caller.  Run `python build_native.py` or call `build()`.
Each source is compiled to its own object file (side by side, and only when it is older than
its source or a header), then the objects are linked.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

HERE = Path(__file__).resolve().parent
ROOT = HERE.parent
SOURCES = [HERE / "csrc" / name
           for name in ("dory_decode.cu", "dory_rotary.cu", "dory_chunk.cu")]
HEADERS = [ROOT / "include" / "dory_decode.h", HERE / "csrc" / "dory_common.h",
           HERE / "csrc" / "dory_sm100.cuh"]
LIBRARY = HERE / "libdory_decode.so"
OBJECTS = HERE / "_build"

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC", "-shared",
    "--cudart", "shared",
]


def nvcc() -> str:
    found = shutil.which("nvcc")
    if found:
        return found
    default = "/usr/local/cuda/bin/nvcc"
    if os.path.exists(default):
        return default
    raise RuntimeError("nvcc not found: the sm_100a library cannot be built")


def _newer(target: Path, inputs) -> bool:
    if not target.exists():
        return False
    built = target.stat().st_mtime
    return all(src.stat().st_mtime <= built for src in inputs)


def up_to_date() -> bool:
    return _newer(LIBRARY, SOURCES + HEADERS)


def _compile(src: Path, force: bool, verbose: bool) -> Path:
    obj = OBJECTS / (src.stem + ".o")
    if not force and _newer(obj, [src, *HEADERS]):
        return obj
    tmp = OBJECTS / f"{src.stem}.{os.getpid()}.tmp.o"
    flags = [f for f in NVCC_FLAGS if f != "-shared"]
    cmd = [nvcc(), *(["-Xptxas=-v"] if verbose else []), *flags, "-I", str(ROOT / "include"),
           "-c", "-o", str(tmp), str(src)]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, obj)
    return obj


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compiles the library if a source is newer than it; returns its path."""
    if not force and up_to_date():
        return LIBRARY
    OBJECTS.mkdir(exist_ok=True)
    with ThreadPoolExecutor(len(SOURCES)) as pool:
        objects = list(pool.map(lambda src: _compile(src, force, verbose), SOURCES))
    tmp = LIBRARY.with_suffix(".so.tmp")
    cmd = [nvcc(), *NVCC_FLAGS, "-o", str(tmp), *map(str, objects)]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, LIBRARY)
    return LIBRARY


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(LIBRARY)
