"""Functional entry points, signature-compatible with ``liger_fused_linear_cross_entropy`` and
``liger_cross_entropy`` (reference: ``src/liger_kernel/transformers/functional.py:81-121`` and ``:42-78``) and
their result type ``CrossEntropyOutput`` (``:34-39``), plus ``liger_fused_linear_jsd`` (``:124-146``), ``liger_layer_norm``,
``liger_rms_norm`` and ``liger_load_balancing_loss``."""

from dataclasses import dataclass
from typing import Optional

import torch

from ..ops.cross_entropy import LigerCrossEntropyFunction
from ..ops.fused_linear_cross_entropy import LigerFusedLinearCrossEntropyFunction
from ..ops.fused_linear_jsd import LigerFusedLinearJSDFunction
from ..ops.load_balancing_loss import LigerLoadBalancingLossFunction, LoadBalancingOutput
from ..ops.norm import LigerLayerNormFunction, LigerRMSNormFunction


@dataclass
class CrossEntropyOutput:
    loss: torch.Tensor
    z_loss: Optional[torch.Tensor] = None
    token_accuracy: Optional[torch.Tensor] = None
    predicted_tokens: Optional[torch.Tensor] = None


def liger_fused_linear_cross_entropy(
    input,
    weight,
    target,
    bias=None,
    ce_weight=None,
    ignore_index: int = -100,
    lse_square_scale: float = 0.0,
    label_smoothing: float = 0.0,
    reduction: str = "mean",
    softcap: Optional[float] = None,
    return_z_loss: bool = False,
    accum_dtype=None,
    use_token_scaling: bool = False,
    return_token_accuracy: bool = False,
    return_predicted_tokens: bool = False,
):
    loss, z_loss, token_accuracy, predicted_tokens = LigerFusedLinearCrossEntropyFunction.apply(
        input, weight, target, bias, ce_weight, ignore_index, lse_square_scale, label_smoothing, reduction, softcap,
        return_z_loss, accum_dtype, use_token_scaling, return_token_accuracy, return_predicted_tokens,
    )
    if not (return_z_loss or return_token_accuracy or return_predicted_tokens):
        return loss
    return CrossEntropyOutput(loss=loss, z_loss=z_loss, token_accuracy=token_accuracy, predicted_tokens=predicted_tokens)


def liger_cross_entropy(
    input,
    target,
    weight=None,
    size_average=None,
    ignore_index: int = -100,
    reduce=None,
    reduction: str = "mean",
    label_smoothing: float = 0.0,
    lse_square_scale: float = 0.0,
    softcap: Optional[float] = None,
    return_z_loss: bool = False,
    return_token_accuracy: bool = False,
    return_predicted_tokens: bool = False,
):
    """Argument order of ``torch.nn.functional.cross_entropy``; ``size_average`` and ``reduce`` are placeholders."""
    loss, z_loss, token_accuracy, predicted_tokens = LigerCrossEntropyFunction.apply(
        input, target, weight, ignore_index, lse_square_scale, label_smoothing, reduction, softcap, return_z_loss,
        return_token_accuracy, return_predicted_tokens,
    )
    if not (return_z_loss or return_token_accuracy or return_predicted_tokens):
        return loss
    return CrossEntropyOutput(loss=loss, z_loss=z_loss, token_accuracy=token_accuracy, predicted_tokens=predicted_tokens)


def liger_fused_linear_jsd(
    student_input,
    student_weight,
    teacher_input,
    teacher_weight,
    shift_labels=None,
    jsd_beta: float = 0.5,
    ignore_index: int = -100,
    temperature: float = 1.0,
    accum_dtype=None,
):
    return LigerFusedLinearJSDFunction.apply(
        student_input, student_weight, teacher_input, teacher_weight, shift_labels, jsd_beta, ignore_index, temperature,
        accum_dtype,
    )


def liger_layer_norm(X, W=None, B=None, eps: float = 1e-6, offset: float = 0.0):
    """Layer norm over the last dimension: ``(x - mean) * rstd * (offset + W) + B``; ``W`` and ``B`` may be None."""
    return LigerLayerNormFunction.apply(X, W, B, eps, offset)


def liger_rms_norm(X, W=None, eps: float = 1e-6, offset: float = 0.0, casting_mode: str = "llama", in_place: bool = True, row_mode=None):
    """RMSNorm over the last dimension: ``x * rstd * (offset + W)``; ``W`` may be None.  ``in_place`` and ``row_mode`` are
    accepted for the reference's call sites and mean nothing here."""
    return LigerRMSNormFunction.apply(X, W, eps, offset, casting_mode, in_place, row_mode)


def liger_load_balancing_loss(
    gate_logits,
    num_experts: int,
    top_k: int = 2,
    attention_mask=None,
    lse_square_scale: float = 0.0,
    return_z_loss: bool = False,
    return_expert_counts: bool = False,
):
    """``num_experts * sum_e f_e P_e`` over the tokens of all layers: f_e the share of tokens that have expert e among their
    ``top_k`` logits, P_e the mean of its softmax probability; plus ``lse_square_scale`` times the mean of lse^2.

    ``gate_logits``: a tensor ``[..., num_experts]`` or a tuple of them, one per layer, ``attention_mask`` one element per token
    of a layer (0 = padding).  Returns the loss, or a ``LoadBalancingOutput`` when a ``return_*`` flag is set;
    ``expert_counts`` is int64 ``[layers, num_experts]`` (``[num_experts]`` for a single tensor)."""
    single = not isinstance(gate_logits, (tuple, list))
    loss, z_loss, counts = LigerLoadBalancingLossFunction.apply(
        num_experts, top_k, attention_mask, lse_square_scale, *((gate_logits,) if single else gate_logits))
    if not (return_z_loss or return_expert_counts):
        return loss
    return LoadBalancingOutput(loss=loss, z_loss=z_loss if return_z_loss else None,
                               expert_counts=(counts[0] if single else counts) if return_expert_counts else None)
