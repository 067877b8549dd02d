"""``Linear`` and ``LayerNorm``: torch's modules of these names on the package's own kernels.

Both are subclasses of the ``torch.nn`` modules and keep their parameters, initialisation and ``state_dict``; ``forward``
calls ``functional.fused_linear`` / ``functional.layer_norm``. There is no CPU path: a CPU tensor raises.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import nn

from . import functional as qf


class Linear(nn.Linear):
    """``act(x weight^T + bias) + residual`` as one kernel. ``round_grads``: as in ``functional.linear_backward``."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, device=None, dtype=None,
                 activation: str = "none", round_grads: bool = False):
        super().__init__(in_features, out_features, bias=bias, device=device, dtype=dtype)
        qf._activation_code(activation)
        self.activation = activation
        self.round_grads = bool(round_grads)

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        return qf.fused_linear(x, self.weight, self.bias, activation=self.activation, residual=residual,
                               round_grads=self.round_grads)

    def extra_repr(self) -> str:
        return super().extra_repr() + ("" if self.activation == "none" else f", activation={self.activation}")


class LayerNorm(nn.LayerNorm):
    """Layer norm over the last axis."""

    def __init__(self, normalized_shape, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True,
                 device=None, dtype=None):
        super().__init__(normalized_shape, eps=eps, elementwise_affine=elementwise_affine, bias=bias, device=device,
                         dtype=dtype)
        if len(self.normalized_shape) != 1:
            raise NotImplementedError(
                f"normalized_shape {tuple(self.normalized_shape)}: the kernels normalise the last axis")

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.shape[-1:] != tuple(self.normalized_shape):
            raise ValueError(f"x {tuple(x.shape)} does not end in {tuple(self.normalized_shape)}")
        return qf.layer_norm(x, self.weight, self.bias, eps=self.eps)
