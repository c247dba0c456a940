"""``LigerLoadBalancingLoss`` module: the arguments of ``liger_load_balancing_loss`` that stay the same from step to step."""

import torch

from .functional import liger_load_balancing_loss


class LigerLoadBalancingLoss(torch.nn.Module):
    def __init__(self, num_experts: int, top_k: int = 2, lse_square_scale: float = 0.0, return_z_loss: bool = False,
                 return_expert_counts: bool = False):
        super().__init__()
        assert 1 <= top_k <= num_experts, f"top_k must be between 1 and num_experts = {num_experts}. Got: {top_k}"
        self.num_experts = num_experts
        self.top_k = top_k
        self.lse_square_scale = lse_square_scale
        self.return_z_loss = return_z_loss
        self.return_expert_counts = return_expert_counts

    def forward(self, gate_logits, attention_mask=None):
        return liger_load_balancing_loss(gate_logits, self.num_experts, self.top_k, attention_mask, self.lse_square_scale,
                                         self.return_z_loss, self.return_expert_counts)
