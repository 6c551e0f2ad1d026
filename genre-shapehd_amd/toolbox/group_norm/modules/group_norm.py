"""GroupNormAct -- group_norm_act as an nn.Module with the parameters (and state_dict keys) of torch.nn.GroupNorm"""
import torch
from torch import nn

from ..functions import group_norm as _F


class GroupNormAct(nn.Module):
    def __init__(self, num_groups, num_channels, eps=1e-5, affine=True, act="none", slope=0.01, device=None, dtype=None):
        """act: "none", "relu", "leaky_relu" (slope), "silu"; see group_norm_act"""
        super().__init__()
        if num_groups < 1 or num_channels < 1 or num_channels % num_groups:
            raise ValueError("GroupNormAct: %d channels do not split into %d groups" % (num_channels, num_groups))
        self.num_groups, self.num_channels, self.eps, self.affine, self.act, self.slope = num_groups, num_channels, eps, affine, act, slope
        if affine:
            self.weight = nn.Parameter(torch.ones(num_channels, device=device, dtype=dtype))
            self.bias = nn.Parameter(torch.zeros(num_channels, device=device, dtype=dtype))
        else:
            self.register_parameter("weight", None)
            self.register_parameter("bias", None)

    def reset_parameters(self):
        if self.affine:
            nn.init.ones_(self.weight)
            nn.init.zeros_(self.bias)

    def forward(self, x):
        return _F.group_norm_act(x, self.num_groups, self.weight, self.bias, self.eps, self.act, self.slope)

    def extra_repr(self):
        return "%d, %d, eps=%g, affine=%s, act=%s" % (self.num_groups, self.num_channels, self.eps, self.affine, self.act)
