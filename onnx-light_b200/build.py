"""Builds the onnxl_b200 shared library (CUDA kernels + C ABI) for sm_100a.

nvcc compiles each csrc/*.cu for `-gencode arch=compute_100a,code=sm_100a`
(cross-compiles without a GPU) and links them into libonnxl_b200.so next to
this file, with the CUDA runtime linked statically.  csrc/torch_binding.cpp becomes the
Python module _b2torch next to it (g++ against torch's headers).
"""
from __future__ import annotations

import concurrent.futures as cf
import glob
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libonnxl_b200.so")
BINDING = os.path.join(HERE, "_b2torch.so")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")

FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden", "--expt-relaxed-constexpr",
    "-fmad=true", "-Xptxas", "-warn-spills",
]


def _needs(obj: str, src: str) -> bool:
    if not os.path.exists(obj):
        return True
    t = os.path.getmtime(obj)
    deps = [src] + glob.glob(os.path.join(CSRC, "*.cuh")) + [
        os.path.join(HERE, "..", "include", "onnxl_b200.h")]
    return any(os.path.getmtime(d) > t for d in deps if os.path.exists(d))


def _compile(src: str, verbose: bool) -> str:
    obj = os.path.join(BUILD, os.path.basename(src).replace(".cu", ".o"))
    if _needs(obj, src):
        cmd = [NVCC, *FLAGS, "-c", src, "-o", obj]
        if verbose:
            cmd.insert(-4, "-Xptxas=-v")
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed for {src}:\n{r.stdout}\n{r.stderr}")
        if verbose and (r.stdout or r.stderr):
            sys.stderr.write(r.stderr)
    return obj


def _binding() -> None:
    src = os.path.join(CSRC, "torch_binding.cpp")
    if not _needs(BINDING, src):
        return
    import sysconfig

    import torch
    root = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(NVCC))
    includes = [os.path.join(root, "include"), os.path.join(root, "include/torch/csrc/api/include"),
                os.path.join(cuda, "include"), sysconfig.get_paths()["include"]]
    cmd = ["g++", "-shared", "-fPIC", "-O2", "-std=c++17", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *[f"-isystem{i}" for i in includes], src, "-o", BINDING,
           f"-L{os.path.join(root, 'lib')}", f"-L{os.path.join(cuda, 'lib64')}", "-ltorch_python",
           "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda", "-l:libcudart.so.12"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"building {BINDING} failed:\n{r.stdout}\n{r.stderr}")


def build(verbose: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    with cf.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        objs = list(ex.map(lambda s: _compile(s, verbose), srcs))
    if not os.path.exists(LIB) or any(os.path.getmtime(o) > os.path.getmtime(LIB) for o in objs):
        cmd = [NVCC, "-shared", "-gencode", "arch=compute_100a,code=sm_100a", "-o", LIB, *objs,
               "-cudart", "static"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    _binding()
    return LIB


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
