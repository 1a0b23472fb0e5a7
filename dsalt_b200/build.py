"""Builds the C-ABI library ``dsalt_b200/_lib/libdsalt_b200.so`` with nvcc for sm_100a, and torch's side of
the operators of :mod:`dsalt_b200.layers` (``dsalt_b200/_lib/_torch_layers.so``) with g++ against it.

    python -m dsalt_b200.build

The library is compiled in-tree so that it travels with the repository; nothing is
installed. Exact IEEE division/sqrt are required by the width and statistics contract,
so fast-math flags are never used.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
OUT_DIR = os.path.join(HERE, "_lib")
LIB = os.path.join(OUT_DIR, "libdsalt_b200.so")
TORCH_SOURCE = os.path.join(CSRC, "torch_layers.cpp")
TORCH_LIB = os.path.join(OUT_DIR, "_torch_layers.so")
SOURCES = ["capi.cu", "signals.cu", "select.cu", "attn_simt.cu", "attn_tc.cu", "attn_bwd.cu", "attn_train.cu", "peer.cu",
           "slots.cu", "cache_append.cu", "cache_attn.cu", "sample.cu", "pack8.cu", "rope.cu", "ffn.cu", "ffn_tc.cu",
           "ffn_few.cu", "ffn_token.cu"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(cand):
        raise RuntimeError("nvcc not found")
    return cand


def _newer(target: str, deps) -> bool:
    if not os.path.exists(target):
        return False
    t = os.path.getmtime(target)
    return all(os.path.getmtime(d) <= t for d in deps)


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(OUT_DIR, exist_ok=True)
    header = os.path.join(ROOT, "include", "dsalt_b200.h")
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh"))] + [header]
    if force or not _newer(LIB, deps):
        _build_kernels(verbose)
    if force or not _newer(TORCH_LIB, [TORCH_SOURCE, header]) or _noted() != _torch_of():
        _build_torch_side()
    return LIB


def _torch_of() -> str:
    """What torch's side is compiled against: its classes have other layouts in another torch."""
    import torch
    return f"torch {torch.__version__}, C++11 ABI {int(torch._C._GLIBCXX_USE_CXX11_ABI)}, python {sys.version.split()[0]}"


def _noted() -> str:
    try:
        with open(TORCH_LIB + ".torch") as f:
            return f.read()
    except OSError:
        return ""


def _build_torch_side() -> None:
    _run_compiler(TORCH_LIB + ".tmp")
    os.replace(TORCH_LIB + ".tmp", TORCH_LIB)
    with open(TORCH_LIB + ".torch", "w") as f:
        f.write(_torch_of())


def _torch_command(target: str) -> list:
    import sysconfig

    import torch
    from torch.utils.cpp_extension import include_paths, library_paths
    cuda = os.path.dirname(os.path.dirname(nvcc()))
    include = [*include_paths(), sysconfig.get_path("include"), os.path.join(cuda, "include")]
    # the g++ that nvcc takes too: another one may link a C++ library of its own beside torch's
    return [shutil.which("g++") or os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-DTORCH_EXTENSION_NAME=_torch_layers",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *[a for p in include for a in ("-isystem", p)], "-I", os.path.join(ROOT, "include"),
           TORCH_SOURCE, "-o", target, "-L" + OUT_DIR, "-ldsalt_b200", "-Wl,-rpath,$ORIGIN",
           *["-L" + p for p in library_paths()], "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python"]


def _run_compiler(target: str) -> None:
    res = subprocess.run(_torch_command(target), capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError("g++ failed:\n" + res.stderr[-8000:])


def _build_kernels(verbose: bool) -> None:
    cmd = [nvcc(), *ARCH, "-O3", "-lineinfo", "-std=c++17", "-shared", "-Xcompiler", "-fPIC",
           "-I", os.path.join(ROOT, "include"), "-o", LIB + ".tmp"]
    if verbose:
        cmd += ["-Xptxas", "-v"]
    cmd += [os.path.join(CSRC, f) for f in SOURCES]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError("nvcc failed:\n" + res.stderr[-8000:])
    if verbose:
        sys.stderr.write(res.stderr)
    os.replace(LIB + ".tmp", LIB)


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
