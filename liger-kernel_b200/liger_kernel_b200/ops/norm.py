"""Layer norm and RMSNorm over the last dimension.

Call surface of the reference's ``LigerLayerNormFunction`` (``src/liger_kernel/ops/layer_norm.py``) and
``LigerRMSNormFunction`` (``src/liger_kernel/ops/rms_norm.py``) on the CUDA kernels of ``libflce_b200.so``
(``csrc/norm_rows.cuh``); checks, allocation and the autograd node are in the compiled binding (``csrc/torch_ops.cpp``).

* Statistics, products and sums are fp32 whatever the input's type; results are rounded once, to the input's type (weight and
  bias gradients to theirs).  Weight and bias may be fp32 beside 16-bit rows.
* Forward keeps the input and, per row, rstd (and the mean); backward is one pass over the rows and one small reduction, whose
  sums run in a fixed order: the same bits in every run.
* ``in_place`` and ``row_mode`` of the reference's RMSNorm are accepted and mean nothing here: the gradient of the input is
  always a tensor of its own, and the launch shape follows from the row's length.
* Any leading dimensions, any row pitch (a slice of a wider tensor is read where it lies), any length of the last dimension from
  one element.  A gradient of the gradient is refused by autograd, and so are inputs with a forward-mode tangent.
* torch.compile, torch.export and make_fx record the launches as operators; torch.func's grad, vjp and vmap apply.
"""

from .. import _lib
from .._torch_ops import norm

_CASTING_MODES = {"llama": True, "gemma": False}      # whether the normalised value is rounded before it meets the weight


class LigerLayerNormFunction:
    """``apply(X, W, B, eps, offset=0.0)``: ``(x - mean) * rstd * (offset + W) + B``.  ``W`` and ``B`` may be None."""

    @staticmethod
    def apply(X, W, B, eps, offset=0.0):
        return norm(X, W, B, _lib.FLCE_LAYER_NORM, eps, offset, False)


class LigerRMSNormFunction:
    """``apply(X, W, eps, offset=0.0, casting_mode="llama", in_place=True, row_mode=None)``: ``x * rstd * (offset + W)``; ``W``
    may be None.  Casting "llama" rounds ``x * rstd`` to the input's type before it meets the weight, "gemma" does not; the
    reference's "none", which computes in the input's type, is refused."""

    @staticmethod
    def apply(X, W, eps, offset=0.0, casting_mode="llama", in_place=True, row_mode=None):
        if casting_mode not in _CASTING_MODES:
            raise NotImplementedError(f"casting_mode must be one of {sorted(_CASTING_MODES)}. Got: {casting_mode}")
        return norm(X, W, None, _lib.FLCE_RMS_NORM, eps, offset, _CASTING_MODES[casting_mode])
