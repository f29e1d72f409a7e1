"""Build the in-tree shared library ``libmxfp4_b200.so`` for sm_100a.

    python -m mxfp4_b200.build [--force]

One nvcc invocation over csrc/mxfp4_b200.cu (a single translation unit that includes the
kernels); the static CUDA runtime keeps the library independent of torch's runtime copy.  Beside
it the host compiler builds ``_attention.so`` from csrc/attention_binding.cpp, the Python binding of
the attention operators against torch's C++ headers (it holds no kernels and finds the library's
entries at run time).  The library comes first and needs nvcc alone; where torch, its headers, Python's or a
host compiler are missing, the binding is left out, which says so.
"""

from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
import sysconfig

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG_DIR)
CSRC = os.path.join(ROOT, "csrc")
INCLUDE = os.path.join(os.path.dirname(ROOT), "include")
OUT = os.path.join(PKG_DIR, "libmxfp4_b200.so")
BINDING = os.path.join(CSRC, "attention_binding.cpp")
BINDING_OUT = os.path.join(PKG_DIR, "_attention.so")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-shared", "-Xcompiler", "-fPIC",
    "-Xptxas", "-v",
]


def sources():
    return sorted(
        os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh"))
    ) + [os.path.join(INCLUDE, "mxfp4_b200.h")]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def up_to_date(out: str, of=None) -> bool:
    if not os.path.exists(out):
        return False
    t = os.path.getmtime(out)
    return all(os.path.getmtime(s) <= t for s in of or sources())


def binding_needs() -> list:
    """What build_binding needs and this host does not have."""
    missing = []
    try:
        import torch

        if not os.path.exists(os.path.join(os.path.dirname(torch.__file__), "include", "ATen", "ATen.h")):
            missing.append("torch's C++ headers")
    except ImportError:
        missing.append("torch")
    if not os.path.exists(os.path.join(sysconfig.get_paths()["include"], "Python.h")):
        missing.append("Python.h")
    if not shutil.which(os.environ.get("CXX", "g++")):
        missing.append("a host C++ compiler")
    return missing


def built_for() -> str:
    """The torch and the Python that run here: _attention.so holds this text of those it was compiled against."""
    import torch

    return f"_attention.so for torch {torch.__version__}, C++ ABI {int(torch.compiled_with_cxx11_abi())}, {sysconfig.get_config_var('SOABI')}"


def binding_fits() -> bool:
    """Whether the _attention.so that is there was compiled against the torch and the Python that run here."""
    with open(BINDING_OUT, "rb") as f:
        return built_for().encode() + b"\0" in f.read()


def build_binding(force: bool = False) -> str:
    """_attention.so; torch's own libraries are already loaded when it is imported."""
    if not force and up_to_date(BINDING_OUT, (BINDING, os.path.join(INCLUDE, "mxfp4_b200.h"))) and binding_fits():
        return BINDING_OUT
    import torch

    home = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(nvcc()))
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", f'-DMXFP4_BUILT_FOR="{built_for()}"',
           "-isystem", os.path.join(home, "include"), "-isystem", os.path.join(home, "include", "torch", "csrc", "api", "include"),
           "-isystem", os.path.join(cuda, "include"), "-isystem", sysconfig.get_paths()["include"],
           "-o", BINDING_OUT + ".tmp", BINDING,
           "-L" + os.path.join(home, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError("the host compiler failed building _attention.so")
    os.replace(BINDING_OUT + ".tmp", BINDING_OUT)
    return BINDING_OUT


def build(force: bool = False, verbose: bool = False) -> str:
    if force or not up_to_date(OUT):
        build_library(verbose)
    missing = binding_needs()
    if missing:
        sys.stderr.write(f"_attention.so is not built, without {', '.join(missing)}: the attention operators need it in Python\n")
    else:
        build_binding(force)
    return OUT


def build_library(verbose: bool = False) -> str:
    cmd = [nvcc(), *NVCC_FLAGS, "-o", OUT + ".tmp", os.path.join(CSRC, "mxfp4_b200.cu")]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError("nvcc failed building libmxfp4_b200.so")
    if verbose:
        sys.stderr.write(r.stderr)
    os.replace(OUT + ".tmp", OUT)
    return OUT


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-v", "--verbose", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, verbose=a.verbose))
