"""Group norm with an activation between the layers of a KAN stack.

A spline layer sees its inputs only inside the range of its knots; in a deep stack the hidden values leave it.
:class:`GroupNormAct` brings the values of each point back to a fixed scale, and with ``tanh`` into (-1, 1), the default
range of the knots.  It works point by point (no batch statistics), so it goes with the physics-informed training step,
where the derivatives of the output with respect to a point are taken through it (``forward_jet``).
"""
from __future__ import annotations

from typing import Optional

import torch

from . import functional as K

__all__ = ["GroupNormAct"]


def _norm_act_kind(module: torch.nn.Module) -> Optional[int]:
    """Kernel id of an activation, or None when the norm's kernels do not know it."""
    kinds = {torch.nn.Identity: K.ACT_IDENTITY, torch.nn.SiLU: K.ACT_SILU, torch.nn.Tanh: K.ACT_TANH}
    return kinds.get(type(module))


class GroupNormAct(torch.nn.Module):
    """``activation(group_norm(x) * weight + bias)`` on ``[N, ..., channels]``, channels last.

    The statistics of a group run over all positions of a sample (the dimensions between the first and the last) and the
    group's channels.  ``activation`` is a module class; Identity, SiLU and Tanh run inside the kernel, any other one
    after it (``forward`` only)."""

    def __init__(self, groups: int, channels: int, eps: float = 1e-5, affine: bool = True,
                 activation=torch.nn.Identity):
        super().__init__()
        if groups < 1 or channels < 1 or channels % groups:
            raise ValueError(f"pde_amd: {channels} channels do not divide into {groups} groups")
        self.groups, self.channels, self.eps, self.affine = groups, channels, eps, affine
        self.activation = activation()
        if affine:
            self.weight = torch.nn.Parameter(torch.ones(channels))
            self.bias = torch.nn.Parameter(torch.zeros(channels))
        else:
            self.register_parameter("weight", None)
            self.register_parameter("bias", None)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        assert x.size(-1) == self.channels
        kind = _norm_act_kind(self.activation)
        y = K.group_norm_act(x, self.groups, self.weight, self.bias, self.eps, K.ACT_IDENTITY if kind is None else kind)
        return self.activation(y) if kind is None else y

    def forward_jet(self, x_jet: torch.Tensor, n_dir: int, n_second: int) -> torch.Tensor:
        """The norm of points on their jets ``[N, channels, 1 + n_dir + n_second]``."""
        kind = _norm_act_kind(self.activation)
        if kind is None:
            raise NotImplementedError("forward_jet supports Identity, SiLU and Tanh activations")
        return K.group_norm_act_jet(x_jet, self.groups, self.weight, self.bias, self.eps, kind, n_dir, n_second)

    def extra_repr(self) -> str:
        return f"{self.groups}, {self.channels}, eps={self.eps}, affine={self.affine}"
