"""Layer norm and RMSNorm over the last dimension, host side.

Call surface of the reference's ``LigerLayerNormFunction`` (``src/liger_kernel/ops/layer_norm.py``) and
``LigerRMSNormFunction`` (``src/liger_kernel/ops/rms_norm.py``) on the CUDA kernels of ``libflce_b200.so``
(``csrc/norm_rows.cuh``).

* Statistics, products and sums are fp32 whatever the input's type; results are rounded once, to the input's type (weight and
  bias gradients to theirs).  Weight and bias may be fp32 beside 16-bit rows.
* Forward keeps the input and, per row, rstd (and the mean); backward is one pass over the rows and one small reduction, whose
  sums run in a fixed order: the same bits in every run.
* ``in_place`` and ``row_mode`` of the reference's RMSNorm are accepted and mean nothing here: the gradient of the input is
  always a tensor of its own, and the launch shape follows from the row's length.
* Any leading dimensions, any row pitch (a slice of a wider tensor is read where it lies), any length of the last dimension from
  one element.  A gradient of the gradient is refused by autograd (``once_differentiable``).
"""

from __future__ import annotations

import ctypes as C

import torch

from torch.autograd.function import once_differentiable

from .. import _lib
from .._lib import Norm, check, lib
from . import fused_linear_cross_entropy as _fl
from .fused_linear_cross_entropy import _DTYPES

LAYER_NORM, RMS_NORM = _lib.FLCE_LAYER_NORM, _lib.FLCE_RMS_NORM
_CASTING_MODES = {"llama": 1, "gemma": 0}      # whether the normalised value is rounded before it meets the weight


def _rows(t: torch.Tensor, hidden: int) -> torch.Tensor:
    """``t`` as ``[rows, hidden]`` with adjacent elements: a view wherever one exists."""
    if t.dim() != 2:
        t = t.reshape(-1, hidden) if t.numel() else t.new_empty((0, hidden))
    if t.stride(1) != 1 and hidden != 1:
        t = t.contiguous()
    return t


def _parameter(name, t, hidden, device):
    if t is None:
        return None
    if t.dim() != 1 or t.shape[0] != hidden:
        raise ValueError(f"{name} must be [{hidden}], got {tuple(t.shape)}")
    if t.dtype not in _DTYPES:
        raise TypeError(f"unsupported {name} dtype {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the input on {device}")
    return t


class _NormCall:
    """One problem: the operands as the library takes them and its argument struct."""

    __slots__ = ("x", "weight", "bias", "struct", "device", "centered")

    def __init__(self, kind, X, W, B, eps, offset, round_xhat):
        _fl._require_cuda(X)
        if X.dim() == 0 or X.shape[-1] == 0:
            raise ValueError(f"expected [..., H] with H >= 1, got {tuple(X.shape)}")
        if X.dtype not in _DTYPES:
            raise TypeError(f"unsupported dtype {X.dtype}")
        hidden = X.shape[-1]
        device = X.device
        W = _parameter("weight", W, hidden, device)
        B = _parameter("bias", B, hidden, device)
        x = _rows(X.detach(), hidden)
        # the kernels take parameters of the rows' type or fp32, both alike: anything else is widened
        types = {t.dtype for t in (W, B) if t is not None}
        wtype = types.pop() if len(types) == 1 else torch.float32
        if types or wtype != x.dtype:
            wtype = torch.float32
        self.weight = None if W is None else W.detach().to(wtype).contiguous()
        self.bias = None if B is None else B.detach().to(wtype).contiguous()
        self.x, self.device, self.centered = x, device, kind == LAYER_NORM
        self.struct = Norm(x.shape[0], hidden, x.stride(0), kind, _DTYPES[x.dtype], _DTYPES[wtype], round_xhat, eps, offset,
                           x.data_ptr(), 0 if W is None else self.weight.data_ptr(), 0 if B is None else self.bias.data_ptr())


def _forward(call: _NormCall, shape, keep_statistics):
    """y in the shape of the input, and the statistics ([2, rows] fp32: rstd, mean) or None."""
    n = call.x.shape[0]
    y = torch.empty(shape, dtype=call.x.dtype, device=call.device)
    stats = rstd = mean = None
    if keep_statistics:
        stats = torch.empty((2 if call.centered else 1, n), dtype=torch.float32, device=call.device)
        rstd = stats.data_ptr()
        mean = rstd + 4 * n if call.centered else None
    with _fl._device_guard(call.device):
        check(lib.flce_b200_norm_forward(C.byref(call.struct), y.data_ptr(), mean, rstd, _fl._stream(call.device)))
    return y, stats


def _backward(call: _NormCall, dY, stats, need_weight, need_bias):
    hidden = call.x.shape[1]
    n = call.x.shape[0]
    dy = _rows(dY, hidden)
    dx = torch.empty(dY.shape, dtype=call.x.dtype, device=call.device)
    dw = torch.empty_like(call.weight) if need_weight else None
    db = torch.empty_like(call.bias) if need_bias else None
    rstd = stats.data_ptr()
    mean = rstd + 4 * n if call.centered else None
    with _fl._device_guard(call.device):
        workspace, nbytes = None, 0
        if need_weight or need_bias:
            nbytes = lib.flce_b200_norm_workspace_bytes(C.byref(call.struct))
            workspace = torch.empty(nbytes, dtype=torch.uint8, device=call.device)
        check(lib.flce_b200_norm_backward(
            C.byref(call.struct), dy.data_ptr(), dy.stride(0), mean, rstd, dx.data_ptr(), None if dw is None else dw.data_ptr(),
            None if db is None else db.data_ptr(), None if workspace is None else workspace.data_ptr(), nbytes,
            _fl._stream(call.device)))
    return dx, dw, db


class _NormFunction(torch.autograd.Function):
    """What the two public Functions share; ``X, W, B`` are the differentiable inputs."""

    @staticmethod
    def run_forward(ctx, kind, X, W, B, eps, offset, round_xhat):
        call = _NormCall(kind, X, W, B, eps, offset, round_xhat)
        y, stats = _forward(call, X.shape, any(ctx.needs_input_grad))
        ctx.save_for_backward(X, W, B, stats)
        ctx.norm_arguments = (kind, eps, offset, round_xhat)
        return y

    @staticmethod
    def run_backward(ctx, dY, need):
        X, W, B, stats = ctx.saved_tensors
        kind, eps, offset, round_xhat = ctx.norm_arguments
        call = _NormCall(kind, X, W, B, eps, offset, round_xhat)
        dx, dw, db = _backward(call, dY, stats, W is not None and need[1], B is not None and need[2])
        dw = None if dw is None else dw.to(W.dtype)
        db = None if db is None else db.to(B.dtype)
        return (dx if need[0] else None), dw, db


class LigerLayerNormFunction(_NormFunction):
    """``(X, W, B, eps, offset=0.0)``: ``(x - mean) * rstd * (offset + W) + B``.  ``W`` and ``B`` may be None."""

    @staticmethod
    def forward(ctx, X, W, B, eps, offset=0.0):
        return _NormFunction.run_forward(ctx, LAYER_NORM, X, W, B, eps, offset, 0)

    @staticmethod
    @once_differentiable
    def backward(ctx, dY):
        return _NormFunction.run_backward(ctx, dY, ctx.needs_input_grad[:3]) + (None, None)


class LigerRMSNormFunction(_NormFunction):
    """``(X, W, eps, offset=0.0, casting_mode="llama", in_place=True, row_mode=None)``: ``x * rstd * (offset + W)``; ``W`` may
    be None.  Casting "llama" rounds ``x * rstd`` to the input's type before it meets the weight, "gemma" does not."""

    @staticmethod
    def forward(ctx, X, W, eps, offset=0.0, casting_mode="llama", in_place=True, row_mode=None):
        if casting_mode not in _CASTING_MODES:
            raise NotImplementedError(f"casting_mode must be one of {sorted(_CASTING_MODES)}. Got: {casting_mode}")
        return _NormFunction.run_forward(ctx, RMS_NORM, X, W, None, eps, offset, _CASTING_MODES[casting_mode])

    @staticmethod
    @once_differentiable
    def backward(ctx, dY):
        dx, dw, _ = _NormFunction.run_backward(ctx, dY, ctx.needs_input_grad[:2] + (False,))
        return dx, dw, None, None, None, None, None


def layer_norm_forward(X, W, B, eps, offset=0.0):
    """Returns ``(Y, saved)``; ``saved`` feeds ``layer_norm_backward``."""
    call = _NormCall(LAYER_NORM, X, W, B, eps, offset, 0)
    y, stats = _forward(call, X.shape, True)
    return y, (call, stats)


def layer_norm_backward(dY, saved):
    """Returns ``(dX, dW, dB)``, None for a parameter that is not there."""
    call, stats = saved
    return _backward(call, dY, stats, call.weight is not None, call.bias is not None)


def rms_norm_forward(X, W, eps, offset=0.0, casting_mode="llama"):
    """Returns ``(Y, saved)``; ``saved`` feeds ``rms_norm_backward``."""
    if casting_mode not in _CASTING_MODES:
        raise NotImplementedError(f"casting_mode must be one of {sorted(_CASTING_MODES)}. Got: {casting_mode}")
    call = _NormCall(RMS_NORM, X, W, None, eps, offset, _CASTING_MODES[casting_mode])
    y, stats = _forward(call, X.shape, True)
    return y, (call, stats)


def rms_norm_backward(dY, saved):
    """Returns ``(dX, dW)``."""
    call, stats = saved
    return _backward(call, dY, stats, call.weight is not None, False)[:2]
