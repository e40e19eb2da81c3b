"""Builds libmoye_b200.so in-tree (moye.jl_b200/lib/) with nvcc for sm_100a.

Usage: python moye.jl_b200/build.py [--force] [--verbose] [--debug]
Also builds lib/moye_calls.so, the row-group calls' way from Python into the library (host code only, against torch's headers).
nvcc cross-compiles, so this works on a machine without a GPU.  Every source is compiled to its
own object (kept under lib/obj/, rebuilt only when it or a header changed), the objects side by
side, then linked.  `--debug` builds lib/libmoye_b200_debug.so with -DMOYE_DEBUG: the kernels
then check every TMA coordinate, tensor-memory column and stage index on the device and report
a violation through the status word instead of touching memory.
"""
import importlib.util
import os
import re
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIBDIR = os.path.join(HERE, "lib")
OUT = os.path.join(LIBDIR, "libmoye_b200.so")
OUT_CALLS = os.path.join(LIBDIR, "moye_calls.so")
OUT_DEBUG = os.path.join(LIBDIR, "libmoye_b200_debug.so")
SOURCES = ["api.cu", "gemm_sm100.cu", "gemm_single.cu", "gemm_pair.cu", "gemm_wide.cu", "gemm_splitk.cu",
           "gemm_skinny.cu", "copy_sm100.cu", "transpose_sm100.cu", "layout_sm100.cu", "axpby_sm100.cu", "ldsm_sm100.cu",
           "rows_sm100.cu", "gemm_grouped.cu", "gemm_lora.cu", "comm_nccl.cu"]
HEADERS = ["common.h", "ptx.cuh", "gemm_common.cuh", os.path.join("..", "..", "include", "moye_b200.h")]
CFLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC"]


def _newer(path, deps):
    if not os.path.exists(path):
        return True
    t = os.path.getmtime(path)
    return any(os.path.getmtime(d) > t for d in deps)


def calls_built_for():
    """What the compiled module of the row-group calls depends on: it reads tensors by torch's own layout of them."""
    import torch
    return f"torch {torch.__version__} {sys.implementation.cache_tag}"


def calls_marker(library_version, built_for=None):
    """The bytes by which moye_calls.so says what it was built for."""
    return f"moye_calls for {built_for or calls_built_for()}, library {library_version};".encode()


def build_calls(force=False):
    """Compile csrc/calls.cpp, a Python extension module; returns its path."""
    src = os.path.join(CSRC, "calls.cpp")
    with open(os.path.join(CSRC, HEADERS[-1])) as f:
        version = re.search(r"#define MOYE_B200_VERSION (\d+)", f.read()).group(1)
    if os.path.exists(OUT_CALLS):
        with open(OUT_CALLS, "rb") as f:
            force = force or calls_marker(version) not in f.read()
    torch_dir = importlib.util.find_spec("torch").submodule_search_locations[0]
    if not force and not _newer(OUT_CALLS, [src, os.path.join(CSRC, HEADERS[-1]), os.path.join(torch_dir, "version.py"), os.path.abspath(__file__)]):
        return OUT_CALLS
    os.makedirs(LIBDIR, exist_ok=True)
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    include = [os.path.join(torch_dir, "include"), os.path.join(torch_dir, "include", "torch", "csrc", "api", "include"),
               sysconfig.get_path("include"), os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(nvcc))), "include")]
    import torch
    res = subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", f'-DMOYE_BUILT_FOR="{calls_built_for()}"', f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"] +
                         [x for i in include for x in ("-isystem", i)] +
                         [src, "-o", OUT_CALLS, "-L" + os.path.join(torch_dir, "lib"), "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda"],
                         capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("building moye_calls failed")
    return OUT_CALLS


def build(force=False, verbose=False, debug=False):
    """Compile every CUDA source of the library for sm_100a; returns the path of the .so."""
    out = OUT_DEBUG if debug else OUT
    objdir = os.path.join(LIBDIR, "obj_debug" if debug else "obj")
    headers = [os.path.join(CSRC, x) for x in HEADERS] + [os.path.abspath(__file__)]
    srcs = [os.path.join(CSRC, s) for s in SOURCES]
    objs = [os.path.join(objdir, s[:-3] + ".o") for s in SOURCES]
    todo = [(s, o) for s, o in zip(srcs, objs) if force or _newer(o, [s] + headers)]
    if not todo and not _newer(out, objs):
        return out
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        raise RuntimeError("nvcc not found; libmoye_b200 cannot be built")
    os.makedirs(objdir, exist_ok=True)
    flags = CFLAGS + (["-DMOYE_DEBUG"] if debug else []) + (["-Xptxas", "-v"] if verbose else [])

    def compile_one(job):
        src, obj = job
        res = subprocess.run([nvcc] + flags + ["-c", src, "-o", obj], capture_output=True, text=True)
        return src, res

    with ThreadPoolExecutor(max_workers=max(1, min(len(todo), os.cpu_count() or 1))) as pool:
        results = list(pool.map(compile_one, todo))
    failed = False
    for src, res in results:
        if verbose or res.returncode != 0:
            sys.stderr.write(res.stdout + res.stderr)
        failed = failed or res.returncode != 0
    if failed:
        raise RuntimeError("nvcc failed building libmoye_b200")
    # NCCL is not linked: comm_nccl.cu looks the library up at run time, so that the .so loads without it
    res = subprocess.run([nvcc, "-shared", "-o", out] + objs + ["-ldl"], capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("linking libmoye_b200 failed")
    return out


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv, debug="--debug" in sys.argv))
    if importlib.util.find_spec("torch"):  # the library itself needs none
        print(build_calls(force="--force" in sys.argv))
