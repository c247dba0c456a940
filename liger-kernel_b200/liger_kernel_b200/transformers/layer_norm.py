"""``LigerLayerNorm`` module (reference: ``src/liger_kernel/transformers/layer_norm.py``)."""

import torch

from ..ops.norm import LigerLayerNormFunction


class LigerLayerNorm(torch.nn.Module):
    """``bias=False`` keeps a bias of zeros, as the reference does; ``offset`` is added to the weight (1.0 for weights that are
    stored as their distance from one)."""

    def __init__(self, hidden_size, eps=1e-6, bias=False, init_fn="ones", offset=0.0):
        super().__init__()
        assert init_fn in ("ones", "zeros"), f"init_fn must be either 'ones' or 'zeros', got {init_fn}"
        self.hidden_size = hidden_size
        self.eps = eps
        self.offset = offset
        self.weight = torch.nn.Parameter(torch.ones(hidden_size) if init_fn == "ones" else torch.zeros(hidden_size))
        self.bias = torch.nn.Parameter(torch.randn(hidden_size) if bias else torch.zeros(hidden_size))
        self.variance_epsilon = eps

    def forward(self, hidden_states):
        return LigerLayerNormFunction.apply(hidden_states, self.weight, self.bias, self.variance_epsilon, self.offset)

    def extra_repr(self):
        return f"{self.hidden_size}, eps={self.eps}"
