"""Builds the CUDA library in-tree with nvcc for sm_100a, and the row operators' torch calls:

    python -m switchyard_b200.build            # -> switchyard_b200/libswitchyard_b200.so, _rows_torch.so

The library: plain nvcc, no torch headers. Its boundary is a C ABI (include/switchyard_b200.h),
so a build takes seconds and it has no compile-time dependency on PyTorch. The one file that has
(csrc/rows_torch.cpp: autograd nodes over that C ABI) is an extension module of its own, no CUDA code in it."""

import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libswitchyard_b200.so")
ROWS = os.path.join(HERE, "_rows_torch.so")
ROWS_SOURCE = os.path.join(CSRC, "rows_torch.cpp")
HEADER = os.path.join(os.path.dirname(HERE), "include", "switchyard_b200.h")
SOURCES = ["runtime.cu", "route.cu", "sort.cu", "combine.cu", "transport.cu", "gemm.cu", "ep.cu",
           "rows.cu", "quant8.cu", "gemm_fp8.cu"]
FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC",
         "--expt-relaxed-constexpr"]


def nvcc():
    exe = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(exe):
        raise RuntimeError("nvcc not found: the switchyard_b200 CUDA library cannot be built")
    return exe


def _older(built, deps):
    return not os.path.exists(built) or any(os.path.getmtime(d) > os.path.getmtime(built) for d in deps)


def stale():
    return _older(LIB, [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh"))] + [HEADER])


def rows_stale():
    return _older(ROWS, [ROWS_SOURCE, HEADER])


def build_rows():
    """Compile the row operators' extension module, linked to the library beside it."""
    import torch
    base = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(nvcc())))
    include = [os.path.join(base, "include"), os.path.join(base, "include", "torch", "csrc", "api", "include"),
               sysconfig.get_paths()["include"], os.path.join(cuda, "include")]
    new = f"{ROWS}.{os.getpid()}"  # put in place whole: a process that loads it finds the old one or the new one
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *(f"-I{d}" for d in include), ROWS_SOURCE,
           "-o", new, "-L" + os.path.join(base, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python", "-L" + HERE,
           "-l:" + os.path.basename(LIB), "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed on {os.path.basename(ROWS_SOURCE)}:\n{r.stdout}")
    os.replace(new, ROWS)


def build(force=False, verbose=False):
    """Compile every .cu of the package into one shared library, and the extension module over it.
    Returns the library's path."""
    if force or stale():
        build_library(verbose)
    if force or rows_stale():
        build_rows()
    return LIB


def build_library(verbose=False):
    objdir = os.path.join(HERE, "_obj")
    os.makedirs(objdir, exist_ok=True)
    procs = []
    for src in SOURCES:
        obj = os.path.join(objdir, src.replace(".cu", ".o"))
        cmd = [nvcc(), *FLAGS, "-c", os.path.join(CSRC, src), "-o", obj] + (["-Xptxas", "-v"] if verbose else [])
        procs.append((src, obj, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    objs = []
    for src, obj, p in procs:
        out, _ = p.communicate()
        if p.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src}:\n{out}")
        if verbose or out.strip():
            print(f"--- {src}\n{out}", file=sys.stderr)
        objs.append(obj)
    cmd = [nvcc(), "-shared", "-o", LIB, *objs, "-gencode", "arch=compute_100a,code=sm_100a"]
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}")


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
