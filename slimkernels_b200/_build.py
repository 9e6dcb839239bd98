"""In-tree build of the native libraries (sm_100a only).

  lib/libsk_w2a8.so        CUDA kernels + C ABI (include/sk_w2a8.h), built with nvcc, no torch dependency
  lib/libsk_w2a8_torch.so  PyTorch C++ extension that marshals tensors into the C ABI

Both are rebuilt only when a source is newer than the library.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

_PKG = os.path.dirname(os.path.abspath(__file__))
_ROOT = os.path.dirname(_PKG)
_CSRC = os.path.join(_PKG, "csrc")
LIB_DIR = os.path.join(_PKG, "lib")
CUDA_LIB = os.path.join(LIB_DIR, "libsk_w2a8.so")
TORCH_LIB = os.path.join(LIB_DIR, "libsk_w2a8_torch.so")

NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
              "-Xcompiler", "-fPIC", "-shared"]


def _newer(target: str, sources) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(s) > t for s in sources)


def _run(cmd, verbose):
    if verbose:
        print(" ".join(cmd), flush=True)
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"build step failed ({proc.returncode}): {' '.join(cmd)}\n{proc.stdout}\n{proc.stderr}")
    if verbose and proc.stderr.strip():
        print(proc.stderr, file=sys.stderr)


def _nvcc() -> str:
    cand = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "bin", "nvcc")
    return cand if os.path.exists(cand) else (shutil.which("nvcc") or "nvcc")


def build_cuda_lib(force: bool = False, verbose: bool = False, ptxas_info: bool = False) -> str:
    """One object per .cu file (compiled side by side, each only when something it includes is newer), one library."""
    headers = [os.path.join(_CSRC, f) for f in os.listdir(_CSRC) if f.endswith((".cuh", ".h"))] + \
              [os.path.join(_ROOT, "include", f) for f in ("sk_w2a8.h", "sk_fp8.h")]
    units = {"sk_w2a8": [h for h in headers if not os.path.basename(h).startswith(("fp8_", "sk_fp8"))],
             "sk_fp8": [h for h in headers if not os.path.basename(h).startswith("w2a8_")]}
    sources = [os.path.join(_CSRC, unit + ".cu") for unit in units]
    if not force and not _newer(CUDA_LIB, sources + headers):      # (a library may come without its objects, and without nvcc)
        return CUDA_LIB
    os.makedirs(LIB_DIR, exist_ok=True)
    objects, jobs = [], []
    for unit, deps in units.items():
        src, obj = os.path.join(_CSRC, unit + ".cu"), os.path.join(LIB_DIR, unit + ".o")
        objects.append(obj)
        if force or _newer(obj, [src] + deps):
            jobs.append([_nvcc()] + NVCC_FLAGS[:-1] + (["-Xptxas", "-v"] if ptxas_info else []) + ["-c", "-o", obj, src])
    with ThreadPoolExecutor() as pool:
        list(pool.map(lambda cmd: _run(cmd, verbose), jobs))
    if force or jobs or _newer(CUDA_LIB, objects):
        _run([_nvcc()] + NVCC_FLAGS + ["-o", CUDA_LIB] + objects, verbose)
    return CUDA_LIB


def build_torch_ext(force: bool = False, verbose: bool = False) -> str:
    srcs = [os.path.join(_CSRC, f) for f in ("torch_ext.cpp", "torch_fp8.cpp")]
    build_cuda_lib(force=False, verbose=verbose)
    if force or _newer(TORCH_LIB, srcs + [os.path.join(_ROOT, "include", f) for f in ("sk_w2a8.h", "sk_fp8.h")]):
        import torch
        from torch.utils import cpp_extension as ce
        incs = [f"-I{p}" for p in ce.include_paths("cuda")]
        tlib = os.path.join(os.path.dirname(torch.__file__), "lib")
        abi = int(torch._C._GLIBCXX_USE_CXX11_ABI)
        cxx = ["g++", "-O2", "-std=c++17", "-fPIC", f"-D_GLIBCXX_USE_CXX11_ABI={abi}",
               "-DTORCH_API_INCLUDE_EXTENSION_H", "-Wno-deprecated-declarations"] + incs
        objects = [os.path.join(LIB_DIR, os.path.basename(src)[:-4] + ".o") for src in srcs]
        with ThreadPoolExecutor() as pool:
            list(pool.map(lambda so: _run(cxx + ["-c", "-o", so[1], so[0]], verbose), zip(srcs, objects)))
        _run(["g++", "-shared", "-o", TORCH_LIB] + objects +
             [f"-L{LIB_DIR}", "-lsk_w2a8", f"-L{tlib}", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch",
              "-L/usr/local/cuda/lib64", "-lcudart", "-Wl,-rpath,$ORIGIN", f"-Wl,-rpath,{tlib}"], verbose)
    return TORCH_LIB


def build_all(force: bool = False, verbose: bool = False) -> None:
    build_cuda_lib(force, verbose)
    build_torch_ext(force, verbose)


if __name__ == "__main__":
    build_all(force="--force" in sys.argv, verbose=True)
