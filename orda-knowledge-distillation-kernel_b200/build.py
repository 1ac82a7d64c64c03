"""Build ``orda_ce_kernel/liborda_b200.so`` in-tree with nvcc for sm_100a.

    python orda-knowledge-distillation-kernel_b200/build.py [--force]

Rebuilds only when a source under csrc/ or include/ is newer than the library.
"""
from __future__ import annotations

import glob
import os
import shutil
import subprocess
import sys
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(ROOT, "include")
LIB_NAME = "liborda_b200.so"
LIB = os.path.join(HERE, "orda_ce_kernel", LIB_NAME)

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "--expt-relaxed-constexpr",
]


def _nvcc() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(cand):
        raise RuntimeError("nvcc not found")
    return cand


def sources() -> list[str]:
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh"))
                  + glob.glob(os.path.join(INCLUDE, "*.h")))


def needs_build() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    return any(os.path.getmtime(s) > t for s in sources())


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not needs_build():
        return LIB
    nvcc = _nvcc()
    with tempfile.TemporaryDirectory(dir=os.path.dirname(LIB)) as tmp:
        # the translation units compile side by side
        objects, running = [], []
        for unit in sorted(glob.glob(os.path.join(CSRC, "*.cu"))):
            objects.append(os.path.join(tmp, os.path.basename(unit) + ".o"))
            cmd = [nvcc, *NVCC_FLAGS, "-I", INCLUDE, "-I", CSRC, "-c", unit, "-o", objects[-1]]
            if verbose:
                print(" ".join(cmd))
            running.append((cmd, subprocess.Popen(cmd)))
        failed = [cmd for cmd, p in running if p.wait() != 0]
        if failed:
            raise subprocess.CalledProcessError(1, failed[0])
        lib = os.path.join(tmp, LIB_NAME)
        subprocess.run([nvcc, *NVCC_FLAGS, "-shared", "-o", lib, *objects], check=True)
        os.replace(lib, LIB)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
