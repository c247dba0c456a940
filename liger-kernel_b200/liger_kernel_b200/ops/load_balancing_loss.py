"""Load-balancing loss of a mixture-of-experts router, with per-expert token counts and gradients.

The term that the mixture-of-experts decoders of the ``transformers`` library add to the language-model loss, and that the
reference's patched forwards take from there (``src/liger_kernel/transformers/model/mixtral.py:17-167``,
``model/qwen3_moe.py:19-155``): a softmax, a top-k, a one-hot tensor of ``[tokens, top_k, experts]`` and several means, in
elementary operations.  Here it is one read of the logits forward and one read and write backward
(``csrc/router_balance.cuh``; checks and the autograd node in ``csrc/torch_ops.cpp``).

* softmax, sums and the loss are fp32 or wider whatever the logits' type; the loss is fp32.
* equal logits are chosen by index, lowest first.  The choice is made on the logits: probabilities that round to the same value
  stay apart.
* tokens that the mask leaves out (elements equal to 0; any other element keeps its token, as one token) are not read; if it leaves
  none, the loss and all gradients are zero.
* a gradient of the gradient, inputs with a forward-mode tangent and vmap are refused; torch.compile, torch.export and make_fx record
  the launches as operators.
"""

from dataclasses import dataclass
from typing import Optional

import torch

from .._torch_ops import load_balancing_loss


@dataclass
class LoadBalancingOutput:
    loss: torch.Tensor
    z_loss: Optional[torch.Tensor] = None
    expert_counts: Optional[torch.Tensor] = None


class LigerLoadBalancingLossFunction:
    """``apply(num_experts, top_k, attention_mask, lse_square_scale, *gate_logits)`` returns ``(loss, z_loss, counts)``, counts
    ``[layers, num_experts]`` int64; gradients flow from the loss to the logits."""

    @staticmethod
    def apply(num_experts, top_k, attention_mask, lse_square_scale, *gate_logits):
        return load_balancing_loss(gate_logits, num_experts, top_k, attention_mask, lse_square_scale)
