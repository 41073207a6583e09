"""Group norm with an activation as a layer's ``norm`` (``SAGEConv(norm=...)``, R/train/graphsage/pytorch/aggregator_dgl.py:210-215)."""
import torch
from torch import nn

from .. import ops


class GroupNorm(nn.Module):
    """``ops.group_norm`` over the last dimension of ``x`` [B, *spatial, num_channels]; the rows of a layer [n, num_channels]: over the channels of each
    row's groups.  ``activation``: None, 'relu', 'silu' or 'gelu', applied to the result in the same pass (a layer takes its norm behind its own
    activation: leave that one None)."""

    def __init__(self, num_groups, num_channels, eps=1e-5, affine=True, activation=None):
        super().__init__()
        if num_groups < 1 or num_channels < 1 or num_channels % num_groups:
            raise ValueError("GroupNorm: %d channels in %d groups" % (num_channels, num_groups))
        if activation not in ops.ACTIVATIONS:
            raise ValueError("GroupNorm: unknown activation %r (None, 'relu', 'silu', 'gelu')" % (activation,))
        self.num_groups, self.num_channels, self.eps, self.activation = num_groups, num_channels, eps, activation
        self.weight = nn.Parameter(torch.ones(num_channels)) if affine else None
        self.bias = nn.Parameter(torch.zeros(num_channels)) if affine else None

    def forward(self, x):
        if x.shape[-1] != self.num_channels:
            raise ValueError("GroupNorm: %d channels, expected %d" % (x.shape[-1], self.num_channels))
        return ops.group_norm(x, self.num_groups, self.weight, self.bias, self.eps, self.activation)

    def extra_repr(self):
        return "%d, %d, eps=%g, affine=%s, activation=%r" % (self.num_groups, self.num_channels, self.eps, self.weight is not None, self.activation)
