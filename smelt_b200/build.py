"""Build libgpt2q.so in-tree with nvcc for sm_100a.

    python -m smelt_b200.build [--force] [--verbose-ptxas]

Objects go to smelt_b200/_build/, the library to smelt_b200/_lib/libgpt2q.so
(both git-ignored; the .so ships with the source tree to the GPU host). Where torch is
installed, its binding of the operators on device memory (csrc/torch_ops.cpp) becomes
smelt_b200/_lib/gpt2q_torch.so next to it.
"""
from __future__ import annotations

import concurrent.futures
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(ROOT, "include")
BUILD = os.path.join(PKG, "_build")
LIBDIR = os.path.join(PKG, "_lib")
LIB = os.path.join(LIBDIR, "libgpt2q.so")
TORCH_LIB = os.path.join(LIBDIR, "gpt2q_torch.so")

# (those that take longest come first, as they are compiled side by side)
SOURCES = ["paged_tree_tc.cu", "paged_tree_i8.cu", "paged_tree_e4m3.cu", "paged_tree.cu", "paged_attn_i8.cu", "paged_attn_e4m3.cu", "paged_attn.cu", "gemm.cu", "gemm_mma.cu", "logprobs.cu", "kernels.cu", "runtime.cu", "attn_tc.cu", "persistent.cu", "tp.cu", "noalloc.cu", "synth.cpp", "blake3.cpp", "smt.cpp", "backward.cu", "paged.cu", "paged_entries.cu"]
HEADERS = ["common.cuh", "kernels.h", "gemm.h", "gemm_mma.h", "persistent.h", "tp.h", "tcgen05.cuh", "blake3.h", "backward.h", "paged.h", "paged_attn.cuh", "device_op.cuh", "logprobs.h"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    return cand


def _newer(src: list[str], dst: str) -> bool:
    if not os.path.exists(dst):
        return True
    t = os.path.getmtime(dst)
    return any(os.path.exists(s) and os.path.getmtime(s) > t for s in src)


def build(force: bool = False, verbose_ptxas: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    os.makedirs(LIBDIR, exist_ok=True)
    hdrs = [os.path.join(CSRC, h) for h in HEADERS] + [os.path.join(INCLUDE, "gpt2q.h")]
    objs, jobs = [], []
    for s in SOURCES:
        src = os.path.join(CSRC, s)
        obj = os.path.join(BUILD, s + ".o")
        objs.append(obj)
        if not (force or _newer([src, __file__] + hdrs, obj)):
            continue
        cmd = [nvcc(), *ARCH, "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC,-O3",
               "--expt-relaxed-constexpr", "-I", INCLUDE, "-I", CSRC, "-c", src, "-o", obj]
        if verbose_ptxas and s.endswith(".cu"):
            cmd[1:1] = ["-Xptxas", "-v"]
        jobs.append(cmd)

    def compile_one(cmd):
        print("[smelt_b200.build]", " ".join(cmd[-3:]), flush=True)
        subprocess.run(cmd, check=True)

    with concurrent.futures.ThreadPoolExecutor(max(1, min(8, os.cpu_count() or 1))) as pool:
        list(pool.map(compile_one, jobs))
    if force or _newer(objs, LIB):
        cmd = [nvcc(), *ARCH, "-shared", "-o", LIB, *objs, "-ldl", "-lpthread"]
        subprocess.run(cmd, check=True)
    build_torch(force)
    return LIB


def build_torch(force: bool = False) -> str | None:
    """The torch binding; None where torch is not installed."""
    if importlib.util.find_spec("torch") is None:
        return None
    src = os.path.join(CSRC, "torch_ops.cpp")
    if not (force or _newer([src, __file__, os.path.join(INCLUDE, "gpt2q.h")], TORCH_LIB)):
        return TORCH_LIB
    import torch
    from torch.utils import cpp_extension

    cuda = os.path.dirname(os.path.dirname(os.path.realpath(nvcc())))
    libs = os.path.join(os.path.dirname(torch.__file__), "lib")
    include = cpp_extension.include_paths() + [os.path.join(cuda, "include"), sysconfig.get_path("include"), INCLUDE]
    print("[smelt_b200.build]", src, "-o", TORCH_LIB, flush=True)
    # under another name first: a process that has the old one mapped keeps it
    tmp = TORCH_LIB + ".tmp"
    subprocess.run([os.environ.get("CXX", "g++"), "-O2", "-std=c++20", "-fPIC", "-shared", "-w",
                    f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
                    *[x for i in include for x in ("-isystem", i)], src, "-o", tmp, "-L", LIBDIR, "-lgpt2q", "-L", libs,
                    "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python", "-Wl,-rpath,$ORIGIN"], check=True)
    os.replace(tmp, TORCH_LIB)
    return TORCH_LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose_ptxas="--verbose-ptxas" in sys.argv)
    print(LIB)
