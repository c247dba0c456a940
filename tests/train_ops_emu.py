"""The norms' entry points of the library compiled for the host (tests/emu/emu_train_ops.cpp), behind the Python operators:
the operators then run on CPU tensors.  Only the tests use this."""

import contextlib
import ctypes as C
import os
import subprocess

_HERE = os.path.dirname(os.path.abspath(__file__))
_ROOT = os.path.dirname(_HERE)
_CSRC = os.path.join(_ROOT, "liger-kernel_b200", "csrc")
_OUT = os.path.join(_HERE, "emu", "_build", "libflce_train_ops_emu.so")
_CUDA_INCLUDE = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "include")
_SOURCES = [os.path.join(_HERE, "emu", "emu_train_ops.cpp"), os.path.join(_HERE, "emu", "simt_emulation.hpp"),
            os.path.join(_ROOT, "include", "flce_b200.h")]
_lib = None


def load():
    global _lib
    if _lib is not None:
        return _lib
    from liger_kernel_b200 import _lib as real

    sources = _SOURCES + [os.path.join(_CSRC, f) for f in os.listdir(_CSRC)]
    if not os.path.exists(_OUT) or any(os.path.getmtime(s) > os.path.getmtime(_OUT) for s in sources):
        os.makedirs(os.path.dirname(_OUT), exist_ok=True)
        fresh = f"{_OUT}.{os.getpid()}"            # put in place whole: tests may run in several processes
        cmd = ["g++", "-x", "c++", "-std=c++20", "-O1", "-w", "-fPIC", "-shared", "-I", _CUDA_INCLUDE, "-I", _CSRC,
               "-I", os.path.join(_ROOT, "include"), "-o", fresh, _SOURCES[0]]
        done = subprocess.run(cmd, capture_output=True, text=True)
        if done.returncode != 0:
            raise RuntimeError("building the emulation failed:\n" + done.stderr[-4000:])
        os.replace(fresh, _OUT)
    lib = C.CDLL(_OUT)
    for name in real.EXPORTS:
        if hasattr(lib, name):
            fn, of = getattr(lib, name), getattr(real.lib, name)
            fn.argtypes, fn.restype = of.argtypes, of.restype
    _lib = lib
    return lib


@contextlib.contextmanager
def installed():
    """The torch binding calls the emulation and accepts CPU tensors."""
    from liger_kernel_b200 import _lib as real, _torch_ops

    lib = load()
    _torch_ops.bind(_OUT, host_memory=True)
    try:
        yield lib
    finally:
        _torch_ops.bind(real.LIB_PATH)
