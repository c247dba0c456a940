"""Loads the compiled torch binding (``csrc/torch_ops.cpp``: allocation, checks and autograd nodes of the operators that run
many times per step) and points it at the loaded ``libflce_b200.so``.

There is no fallback: where the binding is missing or was built against another torch, the operators in it raise an ImportError
when they are called.  The rest of the package does not need it.
"""

import ctypes as C
import os

import torch

from . import _lib

_HERE = os.path.dirname(os.path.abspath(__file__))
BINDING_PATH = os.path.join(_HERE, "libflce_b200_torch.so")
_BUILD = ("build it with `python liger-kernel_b200/build.py` (g++, the headers of the installed torch). "
          "This package has no CPU or PyTorch fallback.")


def bind(path, host_memory=False):
    """Route the binding to the library at ``path`` (``host_memory``: one that computes on host memory, for tests)."""
    missing = _binding.liger_b200_bind(os.fsencode(path), int(host_memory))
    if missing is not None:
        raise ImportError(missing.decode())


def _load():
    if not os.path.exists(BINDING_PATH):
        raise ImportError(f"{BINDING_PATH} is missing: {_BUILD}")
    with open(BINDING_PATH, "rb") as f:
        if f"liger_b200 built against torch {torch.__version__};".encode() not in f.read():
            raise ImportError(f"{BINDING_PATH} was built against another torch than {torch.__version__}: {_BUILD}")
    try:
        torch.ops.load_library(BINDING_PATH)
        binding = C.CDLL(BINDING_PATH)
    except OSError as e:
        raise ImportError(f"{BINDING_PATH} cannot be loaded ({e}): {_BUILD}") from e
    binding.liger_b200_bind.argtypes = [C.c_char_p, C.c_int]
    binding.liger_b200_bind.restype = C.c_char_p
    return binding


def _describe_to_tracers():
    """What the operators that launch kernels return, for tracers that run without data (torch.compile, torch.export, make_fx)."""
    fake = torch.library.register_fake

    @fake("liger_b200::norm")
    def _(x, weight, bias, kind, eps, offset, round_xhat):
        return x.new_empty(x.shape)

    @fake("liger_b200::_norm_with_statistics")
    def _(x, weight, bias, kind, eps, offset, round_xhat):
        planes = 2 if kind == _lib.FLCE_LAYER_NORM else 1
        return x.new_empty(x.shape), x.new_empty((planes, x.numel() // x.shape[-1]), dtype=torch.float32)

    @fake("liger_b200::_norm_backward")
    def _(grad, x, weight, bias, statistics, kind, eps, offset, round_xhat, need_weight, need_bias):
        return (x.new_empty(x.shape), weight.new_empty(weight.shape) if need_weight else None,
                bias.new_empty(bias.shape) if need_bias else None)

    @fake("liger_b200::_load_balancing_loss")
    def _(logits, num_experts, top_k, attention_mask, lse_square_scale):
        x = logits[0]
        return (x.new_empty((num_experts + 3,), dtype=torch.float32),
                x.new_empty((len(logits), num_experts), dtype=torch.int64))

    @fake("liger_b200::_load_balancing_loss_backward")
    def _(grad, logits, attention_mask, values, num_experts, top_k, lse_square_scale):
        x = logits[0]
        return x.new_empty((len(logits), x.numel() // num_experts, num_experts))


def _refusing(message):
    def refuse(*args):
        raise ImportError(message)

    return refuse


try:
    _binding = _load()
    bind(_lib.LIB_PATH)
except ImportError as e:
    norm = load_balancing_loss = _refusing(str(e))
else:
    _describe_to_tracers()
    norm = torch.ops.liger_b200.norm.default
    load_balancing_loss = torch.ops.liger_b200.load_balancing_loss.default
