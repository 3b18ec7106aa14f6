"""Build the sm_100a shared library ``lib/libpa_b200.so`` in-tree with nvcc.

The library exports the C ABI declared in ``include/paged_attention_b200.h``.
It links only the CUDA runtime (the driver's tensor-map encoder is fetched at
run time through ``cudaGetDriverEntryPoint``), so it loads on a machine
without a GPU and can be built there (nvcc cross-compiles for sm_100a).
``build_host`` compiles the CPython extension ``lib/pa_host.so`` beside it (g++).
"""

from __future__ import annotations

import os
import shutil
import subprocess
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
REPO_DIR = PKG_DIR.parent
CSRC = PKG_DIR / "csrc"
LIB_DIR = PKG_DIR / "lib"
LIB_PATH = LIB_DIR / "libpa_b200.so"

SOURCES = ["pa_capi.cu", "pa_kv_append.cu", "pa_decode_mma.cu", "pa_decode_f32.cu", "pa_static_ws.cu",
           "pa_prefill_mma.cu", "pa_prefill_umma.cu", "pa_prefill_umma2.cu", "pa_decode_ext.cu", "pa_decode_direct.cu",
           "pa_decode_f32_ext.cu", "pa_kv_append8.cu",
           "pa_pages.cu"]
HEADERS = ["pa_common.cuh", "pa_internal.h", "pa_tile_math.cuh", "pa_tile_ext.cuh", "pa_decode_kernel.cuh"]
ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]


HOST_SOURCE = CSRC / "pa_host.cpp"
HOST_PATH = LIB_DIR / "pa_host.so"


def _nvcc() -> str:
    cuda_home = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    cand = Path(cuda_home) / "bin" / "nvcc"
    if cand.exists():
        return str(cand)
    found = shutil.which("nvcc")
    if found is None:
        raise RuntimeError("nvcc not found; set CUDA_HOME")
    return found


def _inputs() -> list[Path]:
    files = [CSRC / s for s in SOURCES] + [CSRC / h for h in HEADERS]
    files.append(REPO_DIR / "include" / "paged_attention_b200.h")
    return files


def is_stale() -> bool:
    if not LIB_PATH.exists():
        return True
    lib_mtime = LIB_PATH.stat().st_mtime
    return any(f.stat().st_mtime > lib_mtime for f in _inputs())


def build_library(force: bool = False, verbose: bool = False, extra_flags: list[str] | None = None) -> Path:
    """Compile every CUDA source into ``lib/libpa_b200.so`` (skipped when up to date)."""
    if not force and not is_stale():
        return LIB_PATH
    LIB_DIR.mkdir(parents=True, exist_ok=True)
    tmp = LIB_PATH.with_suffix(".so.tmp")
    cmd = [
        _nvcc(),
        *ARCH_FLAGS,
        "-O3",
        "-lineinfo",
        "-std=c++17",
        "--threads",
        "0",
        "--expt-relaxed-constexpr",
        "-shared",
        "-Xcompiler",
        "-fPIC,-fvisibility=hidden",
        "-Xcompiler",
        "-Wall",
        f"-I{REPO_DIR / 'include'}",
        *(extra_flags or []),
        *[str(CSRC / s) for s in SOURCES],
        "-o",
        str(tmp),
        "-lcudart",
    ]
    if verbose:
        print(" ".join(cmd))
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"nvcc failed ({proc.returncode}):\n{proc.stdout}\n{proc.stderr}")
    if verbose and (proc.stdout or proc.stderr):
        print(proc.stdout, proc.stderr)
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


def build_host(force: bool = False) -> Path:
    """Compile the host extension ``lib/pa_host.so`` against the installed torch
    and ``libpa_b200.so`` beside it (skipped when up to date)."""
    header = REPO_DIR / "include" / "paged_attention_b200.h"
    if not force and HOST_PATH.exists() and HOST_PATH.stat().st_mtime >= max(HOST_SOURCE.stat().st_mtime,
                                                                             header.stat().st_mtime):
        return HOST_PATH
    import sysconfig

    import torch

    torch_dir = Path(torch.__file__).resolve().parent
    cuda_home = Path(os.environ.get("CUDA_HOME", "/usr/local/cuda"))
    tmp = HOST_PATH.with_suffix(".so.tmp")
    cmd = [
        "g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden", "-Wall",
        f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
        "-isystem", str(torch_dir / "include"), "-isystem", str(torch_dir / "include" / "torch" / "csrc" / "api" / "include"),
        "-isystem", str(cuda_home / "include"), "-isystem", sysconfig.get_paths()["include"],
        str(HOST_SOURCE), "-o", str(tmp),
        f"-L{LIB_DIR}", "-l:libpa_b200.so", f"-L{torch_dir / 'lib'}", "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda",
        "-Wl,-rpath,$ORIGIN", f"-Wl,-rpath,{torch_dir / 'lib'}",
    ]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"g++ failed ({proc.returncode}):\n{proc.stdout}\n{proc.stderr}")
    os.replace(tmp, HOST_PATH)
    return HOST_PATH


if __name__ == "__main__":
    import sys

    path = build_library(force="--force" in sys.argv, verbose=True,
                         extra_flags=["-Xptxas", "-v"] if "--ptxas-v" in sys.argv else None)
    print(path)
    print(build_host(force="--force" in sys.argv))
