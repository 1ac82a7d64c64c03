"""Build ``orda_ce_kernel/liborda_b200.so`` in-tree with nvcc for sm_100a.

    python orda-knowledge-distillation-kernel_b200/build.py [--force]

and ``orda_ce_kernel/_student.so``, the Python binding of the student-step operators, with g++ against the
installed torch (where there is none, the library alone, which C programs link to).

Rebuilds only when a source under csrc/ or include/ is newer than a library; ``--force`` for a binding that was
built against another torch.
"""
from __future__ import annotations

import glob
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(ROOT, "include")
LIB_NAME = "liborda_b200.so"
LIB = os.path.join(HERE, "orda_ce_kernel", LIB_NAME)
BINDING = os.path.join(HERE, "orda_ce_kernel", "_student.so")

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
                  + glob.glob(os.path.join(CSRC, "*.cpp")) + glob.glob(os.path.join(INCLUDE, "*.h")))


def has_torch() -> bool:
    return importlib.util.find_spec("torch") is not None


def needs_build() -> bool:
    outputs = [LIB, BINDING] if has_torch() else [LIB]
    if not all(os.path.exists(o) for o in outputs):
        return True
    t = min(os.path.getmtime(o) for o in outputs)
    return any(os.path.getmtime(s) > t for s in sources())


def _binding_flags() -> tuple[list[str], list[str]]:
    """(compiler, linker) flags of the torch extension."""
    import torch
    from torch.utils import cpp_extension

    cuda = os.path.dirname(os.path.dirname(os.path.realpath(_nvcc())))
    paths = [*cpp_extension.include_paths(), sysconfig.get_paths()["include"], os.path.join(cuda, "include")]
    compile_flags = ["-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-DTORCH_API_INCLUDE_EXTENSION_H",
                     f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I", INCLUDE,
                     *[f for p in dict.fromkeys(paths) for f in ("-isystem", p)]]
    torch_lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    link_flags = ["-L", torch_lib, "-lc10", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-lc10_cuda", "-ltorch_python",
                  "-L", os.path.join(cuda, "lib64"), "-lcudart", f"-l:{LIB_NAME}", "-Wl,-rpath,$ORIGIN",
                  f"-Wl,-rpath,{torch_lib}"]
    return compile_flags, link_flags


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not needs_build():
        return LIB
    nvcc = _nvcc()
    flags = _binding_flags() if has_torch() else None
    with tempfile.TemporaryDirectory(dir=os.path.dirname(LIB)) as tmp:
        # the translation units compile side by side
        objects, running = [], []
        for unit in sorted(glob.glob(os.path.join(CSRC, "*.cu"))):
            objects.append(os.path.join(tmp, os.path.basename(unit) + ".o"))
            cmd = [nvcc, *NVCC_FLAGS, "-I", INCLUDE, "-I", CSRC, "-c", unit, "-o", objects[-1]]
            if verbose:
                print(" ".join(cmd))
            running.append((cmd, subprocess.Popen(cmd)))
        if flags:
            binding_object = os.path.join(tmp, "student_binding.o")
            cmd = ["g++", *flags[0], "-c", os.path.join(CSRC, "student_binding.cpp"), "-o", binding_object]
            if verbose:
                print(" ".join(cmd))
            running.append((cmd, subprocess.Popen(cmd)))
        failed = [cmd for cmd, p in running if p.wait() != 0]
        if failed:
            raise subprocess.CalledProcessError(1, failed[0])
        lib = os.path.join(tmp, LIB_NAME)
        subprocess.run([nvcc, *NVCC_FLAGS, "-shared", "-o", lib, *objects], check=True)
        binding = os.path.join(tmp, "_student.so")
        if flags:
            subprocess.run(["g++", "-shared", "-o", binding, binding_object, "-L", tmp, *flags[1]], check=True)
        os.replace(lib, LIB)
        if flags:
            os.replace(binding, BINDING)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
