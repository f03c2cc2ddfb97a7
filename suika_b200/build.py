"""Build recipe for libsuika_reshard.so (the C ABI declared in include/suika_reshard.h) and _train.so, the
Python module that calls its training-step entries on torch tensors.

Both are compiled in-tree, the library with nvcc for sm_100a only; the resulting .so files sit next to
this file so that they travel with the source tree. `python -m suika_b200.build` rebuilds them.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
REPO_DIR = os.path.dirname(PKG_DIR)
CSRC = os.path.join(PKG_DIR, "csrc")
LIB_NAME = "libsuika_reshard.so"
LIB_PATH = os.path.join(PKG_DIR, LIB_NAME)
SOURCES = [os.path.join(CSRC, f) for f in ("plan.cpp", "act.cpp", "exec.cu", "optim.cu", "embed.cu", "logprob.cu")]
DEPS = SOURCES + [os.path.join(CSRC, "internal.h"), os.path.join(CSRC, "train.cuh"), os.path.join(REPO_DIR, "include", "suika_reshard.h")]

EXT_PATH = os.path.join(PKG_DIR, "_train.so")
EXT_SOURCE = os.path.join(CSRC, "bind.cpp")
EXT_DEPS = [EXT_SOURCE, os.path.join(REPO_DIR, "include", "suika_reshard.h")]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC,-Wall",
    "-shared",
]


def nvcc_path() -> str:
    for cand in (shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: the CUDA toolkit is required to build libsuika_reshard.so")


def _older(path: str, deps) -> bool:
    return not os.path.exists(path) or any(os.path.getmtime(p) > os.path.getmtime(path) for p in deps)


def is_stale() -> bool:
    return _older(LIB_PATH, DEPS) or _older(EXT_PATH, EXT_DEPS)


def extension_command(out: str) -> list:
    """g++ with torch's headers and libraries; the library beside it is found through $ORIGIN."""
    import torch
    from torch.utils.cpp_extension import include_paths
    lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    cuda = os.path.join(os.path.dirname(os.path.dirname(nvcc_path())), "include")
    return ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", EXT_SOURCE, *[f"-I{p}" for p in (*include_paths(), cuda, sysconfig.get_paths()["include"])],
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-L{lib}", "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda",
            f"-L{PKG_DIR}", f"-l:{LIB_NAME}", "-Wl,-rpath,$ORIGIN", "-o", out]


def _run(cmd, out: str, what: str, verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd), flush=True)
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"building {what} failed:\n{proc.stdout}\n{proc.stderr}")
    os.replace(cmd[-1], out)


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile the library and the module if they are missing or older than their sources; return the library's path."""
    if force or _older(LIB_PATH, DEPS):
        _run([nvcc_path(), *NVCC_FLAGS, *SOURCES, "-o", LIB_PATH + ".tmp"], LIB_PATH, LIB_NAME, verbose)
    if force or _older(EXT_PATH, EXT_DEPS):
        _run(extension_command(EXT_PATH + ".tmp"), EXT_PATH, "_train.so", verbose)
    return LIB_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
