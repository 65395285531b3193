"""Build ``libakv_b200.so`` (the C ABI of include/akv_b200.h) for sm_100a.

    python -m akv_b200.build [--force] [--verbose]

Compiles every ``csrc/*.cu`` with nvcc for ``sm_100a`` only and links them
into ``akv_b200/libakv_b200.so`` in the source tree, so the built library
travels with the tree; ``csrc/tensor_fields.cpp`` becomes the CPython module
``_tensor_fields`` beside it (g++, torch's headers), whose file name carries
Python's ABI tag and which is built again for another torch.  ``-Xptxas -v``
output (registers, spills, shared memory) is written to
``akv_b200/_build/ptxas.txt``.
"""

from __future__ import annotations

import os
import subprocess
import sys
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(ROOT, "include")
BUILD = os.path.join(PKG, "_build")
LIB = os.path.join(PKG, "libakv_b200.so")
# CPython module: a tensor's fields in one call
FIELDS = os.path.join(PKG, "_tensor_fields" + sysconfig.get_config_var("EXT_SUFFIX"))
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-Xptxas", "-v",
         "--expt-relaxed-constexpr"]


def sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build_fields(force: bool = False) -> str:
    import torch

    src = os.path.join(CSRC, "tensor_fields.cpp")
    stamp = os.path.join(BUILD, "tensor_fields.txt")  # the torch it was built for
    built_for = ""
    if os.path.exists(stamp):
        with open(stamp) as f:
            built_for = f.read()
    if force or built_for != torch.__version__ or _stale(FIELDS, [src]):
        t = os.path.dirname(torch.__file__)
        lib = os.path.join(t, "lib")
        cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC",
               f'-DAKV_TORCH_VERSION="{torch.__version__}"',
               f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
               "-I", os.path.join(t, "include"),
               "-I", os.path.join(t, "include", "torch", "csrc", "api", "include"),
               "-I", sysconfig.get_paths()["include"], src, "-o", FIELDS,
               "-L", lib, "-ltorch_python", "-ltorch_cpu", "-lc10"]
        subprocess.run(cmd, check=True)
        with open(stamp, "w") as f:
            f.write(torch.__version__)
    return FIELDS


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    headers = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    headers.append(os.path.join(INCLUDE, "akv_b200.h"))
    objects, logs = [], []
    for src in sources():
        obj = os.path.join(BUILD, os.path.basename(src)[:-3] + ".o")
        objects.append(obj)
        if force or _stale(obj, [src] + headers):
            cmd = [NVCC, *ARCH, *FLAGS, "-I", INCLUDE, "-I", CSRC, "-c", src, "-o", obj]
            res = subprocess.run(cmd, capture_output=True, text=True)
            logs.append(f"== {os.path.basename(src)}\n{res.stderr}")
            if res.returncode != 0:
                sys.stderr.write(res.stderr)
                raise RuntimeError(f"nvcc failed on {src}")
            if verbose:
                sys.stderr.write(res.stderr)
    if logs:
        with open(os.path.join(BUILD, "ptxas.txt"), "w") as f:
            f.write("\n".join(logs))
    if force or _stale(LIB, objects):
        cmd = [NVCC, *ARCH, "-shared", "-o", LIB, *objects, "-lcudart"]
        subprocess.run(cmd, check=True)
    build_fields(force)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
