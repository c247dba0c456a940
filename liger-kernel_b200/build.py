"""Build libflce_b200.so (the C-ABI CUDA library) in-tree with nvcc for sm_100a, and libflce_b200_torch.so (the torch binding of
the operators that run many times per step) with g++ against the headers of the installed torch.

    python liger-kernel_b200/build.py [--force] [--verbose]

nvcc cross-compiles, so no GPU is needed to build.
"""

import argparse
import importlib.util
import os
import runpy
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "liger_kernel_b200", "libflce_b200.so")
SOURCES = [os.path.join(CSRC, name) for name in ("flce_b200.cu", "norm_b200.cu", "balance_b200.cu")]
BINDING = os.path.join(HERE, "liger_kernel_b200", "libflce_b200_torch.so")
BINDING_SOURCE = os.path.join(CSRC, "torch_ops.cpp")


def _deps():
    deps = [os.path.join(ROOT, "include", "flce_b200.h")]
    for name in sorted(os.listdir(CSRC)):
        deps.append(os.path.join(CSRC, name))
    return deps


def _torch_dir():
    return os.path.dirname(importlib.util.find_spec("torch").origin)


def _torch_version():
    return runpy.run_path(os.path.join(_torch_dir(), "version.py"))["__version__"]


def needs_build():
    if not (os.path.exists(OUT) and os.path.exists(BINDING)):
        return True
    with open(BINDING, "rb") as f:
        if f"liger_b200 built against torch {_torch_version()};".encode() not in f.read():
            return True
    built = min(os.path.getmtime(OUT), os.path.getmtime(BINDING))
    return any(os.path.getmtime(d) > built for d in _deps())


TRACE_OUT = os.path.join(HERE, "liger_kernel_b200", "libflce_b200_trace.so")


def build(force=False, verbose=False, trace=False):
    """trace=True builds a second library with -DFLCE_CLOCK_TRACE: the three warp roles of the main loop count the cycles
    they spend waiting on each barrier (read back with flce_b200_debug_clock_trace; used by bench_gemm.py --trace)."""
    out = TRACE_OUT if trace else OUT
    if not trace and not force and not needs_build():
        return OUT
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    cmd = [
        nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-lineinfo", "-std=c++17",
        "--threads", "0",   # one compiler per source file
        "-shared", "-Xcompiler", "-fPIC", "-I", os.path.join(ROOT, "include"), "-I", CSRC,
        "-o", out,
    ] + (["-DFLCE_CLOCK_TRACE"] if trace else []) + SOURCES
    if verbose:
        cmd.insert(1, "-Xptxas")
        cmd.insert(2, "-v")
    binding = None if trace else subprocess.Popen(_binding_command(nvcc))
    try:
        subprocess.run(cmd, check=True)
    finally:
        status = 0 if binding is None else binding.wait()
    if status != 0:
        raise RuntimeError(f"building {BINDING} failed with exit code {status}")
    return out


def _binding_command(nvcc):
    torch_dir = _torch_dir()
    cuda_dir = os.environ.get("CUDA_HOME") or os.path.dirname(os.path.dirname(os.path.realpath(nvcc)))
    include = [os.path.join(torch_dir, "include"), os.path.join(torch_dir, "include", "torch", "csrc", "api", "include"),
               os.path.join(cuda_dir, "include"), os.path.join(ROOT, "include")]
    return (["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f'-DLIGER_TORCH_VERSION="{_torch_version()}"'] + [f"-I{d}" for d in include] + ["-o", BINDING, BINDING_SOURCE]
            + [f"-L{os.path.join(torch_dir, 'lib')}", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ldl"])


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    ap.add_argument("--trace", action="store_true", help="also build libflce_b200_trace.so (cycle accounting in the main loop)")
    a = ap.parse_args()
    print(build(force=a.force, verbose=a.verbose))
    if a.trace:
        print(build(force=True, verbose=a.verbose, trace=True))
    sys.exit(0)
