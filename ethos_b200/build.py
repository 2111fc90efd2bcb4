"""Build the sm_100a shared library ``ethos_b200/libethos_b200.so`` in tree,
and ``ethos_b200/_training.so``, the autograd nodes of the training operators
over it (C++ against torch's headers; no device code).

    python -m ethos_b200.build          # or: from ethos_b200.build import build; build()

nvcc cross-compiles for sm_100a without a GPU, so this runs on any host with
CUDA 12.9.  The library is rebuilt when a source or header is newer than it.
"""

import os
import shutil
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(ROOT, "include")
LIB_NAME = "libethos_b200.so"
LIB_PATH = os.path.join(PKG, LIB_NAME)
BINDING_SRC = os.path.join(CSRC, "training_torch.cpp")
BINDING_PATH = os.path.join(PKG, "_training.so")

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc_path():
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    return cand


def _sources():
    srcs, deps = [], []
    for name in sorted(os.listdir(CSRC)):
        p = os.path.join(CSRC, name)
        if name.endswith(".cu"):
            srcs.append(p)
        if name.endswith((".cu", ".cuh", ".h")):
            deps.append(p)
    for name in sorted(os.listdir(INCLUDE)):
        deps.append(os.path.join(INCLUDE, name))
    return srcs, deps


def needs_build(out=LIB_PATH):
    if not os.path.exists(out):
        return True
    mtime = os.path.getmtime(out)
    _, deps = _sources()
    return any(os.path.getmtime(d) > mtime for d in deps)


def _build_binding(force, verbose):
    header = os.path.join(INCLUDE, "ethos_b200.h")
    if not force and os.path.exists(BINDING_PATH) and os.path.getmtime(BINDING_PATH) > max(
            os.path.getmtime(BINDING_SRC), os.path.getmtime(header)):
        return
    import sysconfig

    import torch
    home = os.path.dirname(torch.__file__)
    dirs = [os.path.join(home, "include"), os.path.join(home, "include", "torch", "csrc", "api", "include"),
            sysconfig.get_paths()["include"]]
    libdir, tmp = os.path.join(home, "lib"), BINDING_PATH + ".tmp"
    # through nvcc: the host compiler of the library, with libstdc++ shared as torch has it (a $CXX that links its
    # own copy makes the first number in an error message crash)
    cmd = [nvcc_path(), "-O2", "-std=c++17", "--shared", "--cudart", "none", "-Xcompiler", "-fPIC",
           "-DTORCH_EXTENSION_NAME=_training", "-DTORCH_API_INCLUDE_EXTENSION_H",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I", INCLUDE,
           *(f for d in dirs for f in ("-isystem", d)), BINDING_SRC, "-o", tmp, "-L", libdir, "-lc10", "-lc10_cuda",
           "-ltorch_cpu", "-ltorch_python"]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("nvcc failed building %s" % os.path.basename(BINDING_PATH))
    os.replace(tmp, BINDING_PATH)


def build(force=False, verbose=False, extra_flags=()):
    """Compile every ``csrc/*.cu`` into one shared library (sm_100a only), and
    the training operators' binding."""
    _build_library(force, verbose, extra_flags)
    _build_binding(force, verbose)
    return LIB_PATH


def _build_library(force, verbose, extra_flags):
    if not force and not needs_build():
        return
    srcs, _ = _sources()
    tmp = LIB_PATH + ".tmp"
    cmd = [nvcc_path(), *ARCH_FLAGS, "-O3", "-lineinfo", "-std=c++17", "--shared",
           "-Xcompiler", "-fPIC,-O3", "-I", INCLUDE, "-I", CSRC,
           "--expt-relaxed-constexpr", "--threads", "0", *extra_flags, "-o", tmp, *srcs]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("nvcc failed building %s" % LIB_NAME)
    if verbose and (res.stdout or res.stderr):
        sys.stderr.write(res.stdout + res.stderr)
    os.replace(tmp, LIB_PATH)


if __name__ == "__main__":
    force = "--force" in sys.argv
    verbose = "-v" in sys.argv or "--verbose" in sys.argv
    extra = ["-Xptxas", "-v"] if "--ptxas-v" in sys.argv else []
    print(build(force=force, verbose=verbose or bool(extra), extra_flags=extra))
