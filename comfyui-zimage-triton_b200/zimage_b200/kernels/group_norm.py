"""Group normalisation with an activation on sm_100a, channels last, forward and backward."""

from __future__ import annotations

import torch

from .. import _lib

ACTIVATIONS = {"none": 0, "silu": 1}


def group_norm_act(x: torch.Tensor, num_groups: int, weight: torch.Tensor | None = None,
                   bias: torch.Tensor | None = None, eps: float = 1e-6, activation: str = "silu") -> torch.Tensor:
    """act((x - mean) / sqrt(var + eps) * weight + bias) over groups of the last dimension.

    x [B, ..., C] (bf16, fp16, fp32; channels last, C <= 8192, any strides of the others); the mean and the
    variance of a batch entry's group run over its C / num_groups channels and every position
    between.  A convolution's [B, C, H, W] tensor in channels-last memory format is passed as
    ``x.permute(0, 2, 3, 1)`` without a copy.  weight, bias: [C] of one type (bf16, fp16, fp32),
    each may be None.  ``activation``: "silu" or "none".  Returns a contiguous tensor of x's shape
    and type; differentiable in x, weight and bias.
    """
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {tuple(ACTIVATIONS)}, got {activation!r}")
    return _lib.ops().group_norm_act(x, num_groups, weight, bias, eps, act)


class GroupNormAct(torch.nn.Module):
    """``group_norm_act`` with its parameters; the names of ``torch.nn.GroupNorm``."""

    def __init__(self, num_groups: int, num_channels: int, eps: float = 1e-6, affine: bool = True,
                 activation: str = "silu", device=None, dtype=None) -> None:
        super().__init__()
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation must be one of {tuple(ACTIVATIONS)}, got {activation!r}")
        if num_groups < 1 or num_channels % num_groups:
            raise ValueError(f"{num_channels} channels do not split into {num_groups} groups")
        self.num_groups, self.num_channels, self.eps, self.activation = num_groups, num_channels, eps, activation
        kw = dict(device=device, dtype=dtype)
        if affine:
            self.weight = torch.nn.Parameter(torch.ones(num_channels, **kw))
            self.bias = torch.nn.Parameter(torch.zeros(num_channels, **kw))
        else:
            self.register_parameter("weight", None)
            self.register_parameter("bias", None)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return group_norm_act(x, self.num_groups, self.weight, self.bias, self.eps, self.activation)

    def extra_repr(self) -> str:
        return f"{self.num_groups}, {self.num_channels}, eps={self.eps}, activation={self.activation}"
