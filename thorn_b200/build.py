"""Build the sm_100a shared library ``thorn_b200/_lib/libthorn_b200.so`` with nvcc, and the
host extension ``thorn_b200/_lib/thorn_b200_host.*.so`` (``csrc/host_records.cpp``) with g++.

Usage: ``python -m thorn_b200.build [--force]``.  Both are built in-tree so they
travel with the checkout; each is rebuilt when a source or header is newer.  The
library, which is all that users of the C ABI need, comes first.  The extension's
file is named by the torch and Python that it is compiled against: it reads
libtorch's objects, and one of another version must not be loaded.
"""
from __future__ import annotations

import glob
import os
import shutil
import subprocess
import sys
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(ROOT, "include")
LIB_DIR = os.path.join(PKG, "_lib")
LIB = os.path.join(LIB_DIR, "libthorn_b200.so")
HOST_SRC = os.path.join(CSRC, "host_records.cpp")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
    "--expt-relaxed-constexpr",
]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: the thorn_b200 CUDA library cannot be built")


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _stale() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    deps = sources() + glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(INCLUDE, "*.h"))
    return any(os.path.getmtime(d) > t for d in deps)


def host_lib() -> str:
    """The host extension's file for this torch and Python."""
    import torch

    return os.path.join(LIB_DIR, f"thorn_b200_host.torch-{torch.__version__}.{sysconfig.get_config_var('SOABI')}.so")


HOST_LIB = host_lib()


def build_host(force: bool = False, verbose: bool = False) -> str:
    """The CPython extension over this interpreter's libtorch."""
    if not force and os.path.exists(HOST_LIB) and os.path.getmtime(HOST_LIB) >= os.path.getmtime(HOST_SRC):
        return HOST_LIB
    import torch

    os.makedirs(LIB_DIR, exist_ok=True)
    root = os.path.dirname(torch.__file__)
    tmp = f"{HOST_LIB}.{os.getpid()}.tmp"
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-shared",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
           "-I", os.path.join(root, "include"), "-I", os.path.join(root, "include", "torch", "csrc", "api", "include"),
           "-I", sysconfig.get_paths()["include"], HOST_SRC, "-L", os.path.join(root, "lib"), "-ltorch_python",
           "-ltorch_cpu", "-lc10", "-o", tmp]
    if verbose:
        print(" ".join(cmd))
    subprocess.run(cmd, check=True)
    os.replace(tmp, HOST_LIB)
    return HOST_LIB


def build_library(force: bool = False, verbose: bool = False) -> str:
    """The CUDA library."""
    if not force and not _stale():
        return LIB
    os.makedirs(LIB_DIR, exist_ok=True)
    nvcc = _nvcc()
    objs = []
    for src in sources():
        obj = os.path.join(LIB_DIR, os.path.basename(src).replace(".cu", ".o"))
        cmd = [nvcc, *NVCC_FLAGS, "-I", INCLUDE, "-I", CSRC, "-c", src, "-o", obj]
        if verbose:
            print(" ".join(cmd))
        subprocess.run(cmd, check=True)
        objs.append(obj)
    tmp = LIB + ".tmp"
    cmd = [nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-Xcompiler", "-fPIC", *objs, "-o", tmp]
    subprocess.run(cmd, check=True)
    os.replace(tmp, LIB)
    for o in objs:
        os.remove(o)
    return LIB


def build(force: bool = False, verbose: bool = False) -> str:
    """Both; returns the library's path."""
    lib = build_library(force, verbose)
    build_host(force, verbose)
    return lib


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
