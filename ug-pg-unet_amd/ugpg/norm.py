"""Group normalisation with an activation on channels-last activations.

The normalisation of a DoubleConv (``norm="group"``) where a GPU holds too few images for
BatchNorm's batch statistics: a sample's result does not depend on the others, there are no
running statistics to synchronise, and train and eval mode compute the same.  The
reference normalises with BatchNorm2d only (UG_unet_parts.py:11,14).
"""
from __future__ import annotations

import torch
import torch.nn as nn

from . import ops
from ._nodes import nodes


def group_norm_act(x, num_groups, weight=None, bias=None, eps=1e-5, activation="relu"):
    """act(group_norm(x)) of channels-last ``x`` (B, ..., C), float32 or bfloat16.

    Statistics run over a sample's middle dimensions and its C/num_groups consecutive
    channels, in float32.  weight, bias: (C,) float32 or None.  activation: "relu", "silu"
    or "none".  Differentiable in x, weight and bias (once).  Less than 2^22 groups over the whole
    batch, at most 2^20 channels."""
    if x.dim() < 2:
        raise ValueError(f"group_norm_act: expected (B, ..., C), got shape {tuple(x.shape)}")
    c = x.shape[-1]
    if not isinstance(num_groups, int) or num_groups < 1 or c % num_groups:
        raise ValueError(f"group_norm_act: {c} channels do not divide into {num_groups} groups")
    if activation not in ops.ACTIVATIONS:
        raise ValueError(f"group_norm_act: activation must be one of {tuple(ops.ACTIVATIONS)}, "
                         f"got {activation!r}")
    if not eps >= 0.0:
        raise ValueError(f"group_norm_act: eps must not be negative, got {eps}")
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"group_norm_act: x must be float32 or bfloat16, got {x.dtype}")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if tuple(p.shape) != (c,):
            raise ValueError(f"group_norm_act: {name} must have shape ({c},), got {tuple(p.shape)}")
        if p.dtype != torch.float32:
            raise TypeError(f"group_norm_act: {name} must be float32, got {p.dtype}")
        if p.device != x.device:
            raise RuntimeError(f"group_norm_act: {name} is on {p.device}, x on {x.device}")
    if x.numel() == 0:
        raise ValueError(f"group_norm_act: empty input {tuple(x.shape)}")
    if x.shape[0] * num_groups >= 1 << 22:
        raise ValueError(f"group_norm_act: {x.shape[0]} samples of {num_groups} groups are {1 << 22} or more")
    if c > 1 << 20 or x.shape[0] * -(-c // 256) > 1 << 22:
        raise ValueError(f"group_norm_act: {x.shape[0]} samples of {c} channels are too many")
    if not x.is_cuda:
        raise RuntimeError("ugpg: tensor is not on a ROCm/HIP device (no CPU fallback)")
    if not x.is_contiguous():
        x = x.contiguous()
    if weight is not None and not weight.is_contiguous():
        weight = weight.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    return nodes().group_norm_act(x, weight, bias, num_groups, eps, ops.ACTIVATIONS[activation])


class GroupNormAct(nn.GroupNorm):
    """nn.GroupNorm followed by an activation, computed channels last: the group twin of
    BatchNorm2d + ReLU in a DoubleConv.  Parameters and state_dict are nn.GroupNorm's.

    ``forward`` takes and returns (N, C, *spatial) as nn.GroupNorm does; the result is in
    channels_last memory format, and an input already in that format is read as it lies."""

    def __init__(self, num_groups, num_channels, eps=1e-5, affine=True, activation="relu"):
        super().__init__(num_groups, num_channels, eps=eps, affine=affine)
        if activation not in ops.ACTIVATIONS:
            raise ValueError(f"GroupNormAct: activation must be one of {tuple(ops.ACTIVATIONS)}, "
                             f"got {activation!r}")
        self.activation = activation

    def forward(self, x):
        if x.dim() < 2 or x.shape[1] != self.num_channels:
            raise ValueError(f"GroupNormAct: expected (N, {self.num_channels}, *), got "
                             f"{tuple(x.shape)}")
        y = group_norm_act(x.movedim(1, -1), self.num_groups, self.weight, self.bias, self.eps,
                           self.activation)
        return y.movedim(-1, 1)

    def extra_repr(self):
        return f"{super().extra_repr()}, activation={self.activation}"
