"""In-tree build of the native pieces for sm_100a.

    python -m fastforwardattention_b200.build [--force]

  libffa_b200.so       the CUDA kernels behind the C ABI of include/ffa_c_api.h (nvcc)
  ff_attention*.so     the torch extension exposing FastForwardAttn (g++, links the above)

Replaces the reference's setup.py (sm_80/sm_86) and compile.sh (sm_75/80/86): one target
architecture, sm_100a.  Outputs land beside this file so that they are found by relative path.
"""
from __future__ import annotations

import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
CUDA_HOME = os.path.dirname(os.path.dirname(NVCC))
LIB = os.path.join(PKG, "libffa_b200.so")
EXT = os.path.join(PKG, "ff_attention" + (sysconfig.get_config_var("EXT_SUFFIX") or ".so"))

API_HEADER = os.path.join(ROOT, "include", "ffa_c_api.h")
COMMON_HEADERS = ["ffa_internal.h", "ffa_device_common.cuh", "ffa_launch.cuh"]
# every source with the headers it includes: what makes its object stale
CUDA_SOURCES = {
    "ffa_decode_kernels.cu": [*COMMON_HEADERS, "ffa_stream_kernel.cuh", "ffa_prune_kernels.cuh", "ffa_prune_stream_kernel.cuh"],
    "ffa_tree_kernels.cu": [*COMMON_HEADERS, "ffa_tree_kernel.cuh", "ffa_tree_umma_kernel.cuh"],
    "ffa_evict_kernels.cu": COMMON_HEADERS,
    "ffa_beam_kernels.cu": COMMON_HEADERS,
    "ffa_strategies_api.cu": ["ffa_internal.h", "ffa_plan.h", API_HEADER],
    "ffa_tree_api.cu": ["ffa_internal.h", "ffa_plan.h", API_HEADER],
    "ffa_c_api.cu": ["ffa_internal.h", "ffa_plan.h", API_HEADER],
    "ffa_no_alloc.cu": ["ffa_internal.h", API_HEADER],
    "ffa_peer_gather.cu": COMMON_HEADERS,
}
CUDA_DEPS = sorted({*CUDA_SOURCES, *(h for deps in CUDA_SOURCES.values() for h in deps)})
NVCC_FLAGS = ["-O3", "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo",
              "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr"]


def _stale(target: str, deps) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d if os.path.isabs(d) else os.path.join(CSRC, d)) > t for d in deps)


def _run(cmd) -> None:
    print("+", " ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)


def build_library(force: bool = False, verbose_ptxas: bool = False) -> str:
    if force or _stale(LIB, CUDA_DEPS):
        os.makedirs(os.path.join(PKG, "build"), exist_ok=True)
        objs, cmds = [], []
        for src, headers in CUDA_SOURCES.items():
            obj = os.path.join(PKG, "build", src.replace(".cu", ".o"))
            if force or _stale(obj, [src, *headers]):
                cmds.append([NVCC, *NVCC_FLAGS, *(["-Xptxas", "-v"] if verbose_ptxas else []), "-c",
                             os.path.join(CSRC, src), "-o", obj])
            objs.append(obj)
        with ThreadPoolExecutor(max(1, os.cpu_count() or 1)) as pool:
            list(pool.map(_run, cmds))
        _run([NVCC, "-shared", "-gencode", "arch=compute_100a,code=sm_100a", "-o", LIB, *objs])
    return LIB


def build_extension(force: bool = False) -> str:
    src = os.path.join(CSRC, "torch_binding.cpp")
    if force or _stale(EXT, [src, os.path.join(ROOT, "include", "ffa_c_api.h"), LIB]):
        import torch
        from torch.utils.cpp_extension import include_paths

        tlib = os.path.join(os.path.dirname(torch.__file__), "lib")
        inc = [f"-I{p}" for p in include_paths()] + [f"-I{sysconfig.get_paths()['include']}",
                                                     f"-I{CUDA_HOME}/include", f"-I{os.path.join(ROOT, 'include')}"]
        _run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-DTORCH_EXTENSION_NAME=ff_attention",
              "-DTORCH_API_INCLUDE_EXTENSION_H", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
              *inc, src, "-o", EXT, f"-L{PKG}", "-lffa_b200", f"-L{tlib}", "-lc10", "-lc10_cuda", "-ltorch_cpu",
              "-ltorch_cuda", "-ltorch", "-ltorch_python", "-Wl,-rpath,$ORIGIN", f"-Wl,-rpath,{tlib}"])
    return EXT


def build_all(force: bool = False) -> None:
    build_library(force)
    build_extension(force)


if __name__ == "__main__":
    build_all(force="--force" in sys.argv)
