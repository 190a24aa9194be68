"""Build recipe for the sm_100a extension ``thesis_b200/_lib/libeesd.so`` (in-tree).

    python -m thesis_b200.build          # rebuild when a source is newer than the library

The library is a plain C-ABI shared object (``include/eesd.h``) linked against the static
CUDA runtime, so it loads in any process that has the NVIDIA driver (and, for the symbol
checks of the CPU test suite, in a process without one).
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
LIB = PKG / "_lib" / "libeesd.so"
SOURCES = ["gemm_tc.cu", "kernels.cu", "runtime.cu", "head_static.cu", "cache_ops.cu", "attn_tree.cu",
           "attn_tree_tc.cu"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found: the CUDA toolkit is required to build thesis_b200")


def needs_build() -> bool:
    if not LIB.exists():
        return True
    t = LIB.stat().st_mtime
    deps = [CSRC / s for s in SOURCES] + list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.h")) + [ROOT / "include" / "eesd.h"]
    return any(p.stat().st_mtime > t for p in deps)


def build(force: bool = False, verbose: bool = False) -> Path:
    if not force and not needs_build():
        return LIB
    LIB.parent.mkdir(parents=True, exist_ok=True)
    tmp = LIB.with_suffix(".so.tmp")
    flags = [*ARCH, "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC,-O2", "-I", str(ROOT / "include")]
    if verbose:
        flags.insert(0, "-Xptxas=-v")

    def run(cmd):
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True, cwd=str(CSRC))

    with tempfile.TemporaryDirectory() as d, ThreadPoolExecutor(len(SOURCES)) as pool:   # one nvcc per source
        objs = [str(Path(d) / (s + ".o")) for s in SOURCES]
        list(pool.map(lambda so: run([nvcc(), *flags, "-c", str(CSRC / so[0]), "-o", so[1]]), zip(SOURCES, objs)))
        run([nvcc(), *flags, "-shared", "-o", str(tmp), *objs])
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
