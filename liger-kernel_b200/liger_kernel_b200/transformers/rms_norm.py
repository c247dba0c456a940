"""``LigerRMSNorm`` module (reference: ``src/liger_kernel/transformers/rms_norm.py``)."""

import torch

from ..ops.norm import LigerRMSNormFunction


class LigerRMSNorm(torch.nn.Module):
    def __init__(self, hidden_size, eps=1e-6, offset=0.0, casting_mode="llama", init_fn="ones", in_place=True, row_mode=None,
                 elementwise_affine=True):
        super().__init__()
        assert init_fn in ("ones", "zeros"), f"init_fn must be either 'ones' or 'zeros', got {init_fn}"
        if elementwise_affine:
            self.weight = torch.nn.Parameter(torch.ones(hidden_size) if init_fn == "ones" else torch.zeros(hidden_size))
        else:
            self.register_parameter("weight", None)
        self.hidden_size = hidden_size
        self.variance_epsilon, self.offset, self.casting_mode = eps, offset, casting_mode
        self.in_place, self.row_mode = in_place, row_mode

    def forward(self, hidden_states):
        return LigerRMSNormFunction.apply(hidden_states, self.weight, self.variance_epsilon, self.offset, self.casting_mode,
                                          self.in_place, self.row_mode)

    def extra_repr(self):
        return f"{self.hidden_size}, eps={self.variance_epsilon}, offset={self.offset}, casting_mode={self.casting_mode}"
