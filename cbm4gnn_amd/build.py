"""Build the shared libraries of the package in-tree.

    libcbm_hip.so    hipcc, gfx950 only: the HIP kernels and their C-ABI launchers
    libcbm_host.so   g++ / OpenMP: the host-side format builder
    cbm_autograd.so  g++ against torch, where it is installed: the dense operators' autograd nodes, over libcbm_hip.so

Run ``python -m cbm4gnn_amd.build`` (no GPU needed: hipcc cross-compiles).  The reference builds
its extension with cmake + setuptools against MKL and arbok (``cbm/setup.py:15-47``); none of
that applies here.
"""
from __future__ import annotations

import importlib.util
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
REPO_DIR = os.path.dirname(PKG_DIR)
SRC_DIR = os.path.join(PKG_DIR, "csrc")
LIB_DIR = os.path.join(PKG_DIR, "lib")
HIP_LIB = os.path.join(LIB_DIR, "libcbm_hip.so")
HOST_LIB = os.path.join(LIB_DIR, "libcbm_host.so")
AUTOGRAD_LIB = os.path.join(LIB_DIR, "cbm_autograd.so")

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

HIP_FLAGS = [
    "-O3", "--offload-arch=gfx950", "-fPIC", "-std=c++17",
    "-ffp-contract=off",                       # FMAs are written explicitly where they are meant
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
]
HOST_FLAGS = ["-O3", "-fopenmp", "-shared", "-fPIC", "-std=c++17", "-Wall"]


def _run(cmd):
    proc = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    out = "\n".join(l for l in proc.stdout.splitlines() if "packed-fp32-ops' is not a recognized feature" not in l)
    if proc.returncode != 0:
        raise RuntimeError(f"build failed ({proc.returncode}): {' '.join(cmd)}\n{out}")
    return out


HIP_SOURCES = ["cbm_kernels.hip", "norm_kernels.hip", "label_kernels.hip", "ortho_kernels.hip"]


def build_hip(verbose: bool = False) -> str:
    os.makedirs(LIB_DIR, exist_ok=True)
    # one object per source, side by side, then the library
    objects = [os.path.join(LIB_DIR, name.replace(".hip", ".o")) for name in HIP_SOURCES]
    with ThreadPoolExecutor(len(HIP_SOURCES)) as pool:
        outs = list(pool.map(lambda so: _run([HIPCC, *HIP_FLAGS, "-c", "-o", so[1], os.path.join(SRC_DIR, so[0])]),
                             zip(HIP_SOURCES, objects)))
    out = "\n".join(o for o in outs + [_run([HIPCC, *HIP_FLAGS, "-shared", "-o", HIP_LIB, *objects])] if o.strip())
    if verbose and out.strip():
        print(out)
    return HIP_LIB


def build_host(verbose: bool = False) -> str:
    os.makedirs(LIB_DIR, exist_ok=True)
    out = _run(["g++", *HOST_FLAGS, "-o", HOST_LIB, os.path.join(SRC_DIR, "cbm_builder.cpp")])
    if verbose and out.strip():
        print(out)
    return HOST_LIB


def _hip_headers() -> str:
    """The include directory of the ROCm that the compiler belongs to, wherever ``HIPCC`` says that is."""
    found = shutil.which(HIPCC)
    roots = [os.path.dirname(os.path.dirname(p)) for p in ((found, os.path.realpath(found)) if found else ())]
    for root in (*roots, os.environ.get("ROCM_PATH", ""), "/opt/rocm"):
        if root and os.path.exists(os.path.join(root, "include", "hip", "hip_runtime_api.h")):
            return os.path.join(root, "include")
    raise RuntimeError(f"no HIP headers beside {HIPCC}, under ROCM_PATH or in /opt/rocm")


def build_autograd(verbose: bool = False) -> str:
    """After ``build_hip``, whose library it is linked to."""
    import sysconfig

    import torch

    root = os.path.dirname(torch.__file__)
    include, libs = os.path.join(root, "include"), os.path.join(root, "lib")
    out = _run(["g++", "-O2", "-shared", "-fPIC", "-std=c++17", "-Wall", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
                f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
                *(f"-isystem{d}" for d in (include, os.path.join(include, "torch", "csrc", "api", "include"),
                                           sysconfig.get_paths()["include"], _hip_headers())),
                "-o", AUTOGRAD_LIB, os.path.join(SRC_DIR, "dense_autograd.cpp"),
                f"-L{LIB_DIR}", "-l:libcbm_hip.so", "-Wl,-rpath,$ORIGIN",
                f"-L{libs}", "-ltorch_python", "-ltorch_cpu", "-ltorch", "-lc10_hip", "-lc10"])
    if verbose and out.strip():
        print(out)
    return AUTOGRAD_LIB


def build_all(verbose: bool = False):
    """The two C-ABI libraries, which need no torch, and, where there is one to compile against, the autograd module
    (``AUTOGRAD_LIB``).  Side by side, but for what is linked to another.  Returns the paths of the first two."""
    with ThreadPoolExecutor(1) as pool:
        pending = pool.submit(build_host, verbose)
        hip = build_hip(verbose)
        host = pending.result()
        if importlib.util.find_spec("torch") is not None:
            build_autograd(verbose)
    return hip, host


if __name__ == "__main__":
    for p in build_all(verbose=True):
        print("built", p)
    if importlib.util.find_spec("torch") is not None:
        print("built", AUTOGRAD_LIB)
    else:
        print("no torch: without", AUTOGRAD_LIB)
    sys.exit(0)
