"""Build the sm_100a C-ABI library ``dsv4attn/libdsv4attn.so`` in-tree.

    python tt-deepseek-v4_b200/build.py [--force] [--verbose]

Compiles every ``csrc/*.cu`` with nvcc for ``sm_100a`` (no PTX for other
architectures, no JIT) and links one shared library against the shared
CUDA runtime, so the process that loads it through ctypes shares one
runtime (and one primary context) with PyTorch.  ``csrc/torch_ops.cpp`` (the
low-bit operators over torch tensors) becomes ``dsv4attn/_torch_ops.so``, a
Python module linked against that library and torch.  Objects are rebuilt
only when a source or header is newer than the library, the module also when
torch or Python is not the one it was built with.
"""

from __future__ import annotations

import argparse
import glob
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")
OUT_DIR = os.path.join(HERE, "dsv4attn")
LIB = os.path.join(OUT_DIR, "libdsv4attn.so")
TORCH_SRC = os.path.join(CSRC, "torch_ops.cpp")
TORCH_LIB = os.path.join(OUT_DIR, "_torch_ops.so")
OBJ_DIR = os.path.join(HERE, "_build")

GENCODE = "-gencode=arch=compute_100a,code=sm_100a"
NVCC_FLAGS = ["-O3", "-lineinfo", "-std=c++17", GENCODE, "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
              "-Xptxas", "-warn-spills"]


def find_nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found (set NVCC or add the CUDA toolkit to PATH)")


def _sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _headers():
    return sorted(glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(INCLUDE, "*.h")))


def needs_build() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    return any(os.path.getmtime(p) > t for p in _sources() + _headers() + [__file__])


def build_torch_ops(force: bool = False, verbose: bool = False) -> str:
    """The Python module over torch tensors (needs the library built)."""
    import torch
    deps = [TORCH_SRC, __file__] + glob.glob(os.path.join(INCLUDE, "*.h"))
    # it links torch's C++ internals and the interpreter's
    made_with = f"torch {torch.__version__} abi {int(torch._C._GLIBCXX_USE_CXX11_ABI)} {sysconfig.get_config_var('SOABI')}"
    key = os.path.join(OBJ_DIR, "_torch_ops.key")
    if not force and os.path.exists(TORCH_LIB) and os.path.getmtime(TORCH_LIB) > max(map(os.path.getmtime, deps)) \
            and os.path.exists(key):
        with open(key) as f:
            if f.read() == made_with:
                return TORCH_LIB
    tdir = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(find_nvcc())))
    inc = [os.path.join(tdir, "include"), os.path.join(tdir, "include", "torch", "csrc", "api", "include"),
           os.path.join(cuda, "include"), sysconfig.get_paths()["include"], INCLUDE]
    tmp = TORCH_LIB + ".tmp"
    # the g++ that nvcc compiles the host side with, not $CXX: one that links
    # its own static libstdc++ gives the process a second C++ runtime, and an
    # exception that crosses into torch's ends it
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *(f for i in inc for f in ("-isystem", i)), TORCH_SRC, "-o", tmp, "-L" + OUT_DIR, "-l:libdsv4attn.so",
           "-Wl,-rpath,$ORIGIN", "-L" + os.path.join(tdir, "lib"), "-lc10", "-ltorch_cpu", "-ltorch_cuda", "-ltorch",
           "-ltorch_python", "-lc10_cuda"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, TORCH_LIB)
    os.makedirs(OBJ_DIR, exist_ok=True)
    with open(key, "w") as f:
        f.write(made_with)
    return TORCH_LIB


def build(force: bool = False, verbose: bool = False, ptxas_info: bool = False) -> str:
    if not force and not needs_build():
        build_torch_ops(verbose=verbose)
        return LIB
    nvcc = find_nvcc()
    os.makedirs(OBJ_DIR, exist_ok=True)
    objs = []
    hdr_t = max(os.path.getmtime(p) for p in _headers())
    for src in _sources():
        obj = os.path.join(OBJ_DIR, os.path.basename(src)[:-3] + ".o")
        objs.append(obj)
        if not force and os.path.exists(obj) and os.path.getmtime(obj) > max(os.path.getmtime(src), hdr_t):
            continue
        cmd = [nvcc, *NVCC_FLAGS, "-I", INCLUDE, "-c", src, "-o", obj]
        if ptxas_info:
            cmd[1:1] = ["-Xptxas", "-v"]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
    tmp = LIB + ".tmp"
    cmd = [nvcc, GENCODE, "-shared", "-cudart", "shared", "-o", tmp, *objs]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, LIB)
    build_torch_ops(force=force, verbose=verbose)
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    ap.add_argument("--ptxas-info", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, verbose=a.verbose, ptxas_info=a.ptxas_info))
    sys.exit(0)
