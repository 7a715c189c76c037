"""Group normalisation of channels-last maps fused with a residual and an activation (csrc/group_norm.hip, csrc/autograd.cpp).

The counterpart of ``batch_norm_act`` whose statistics come from one image's group of channels: nothing depends on the
batch, so it serves training at a few images per GPU, and evaluation computes what training computes.  CPU tensors /
``set_backend('torch')`` run plain torch operations.
"""
from __future__ import annotations

import math
from typing import Optional

import torch
import torch.nn as nn

from . import _backend as B

_TYPES = (torch.bfloat16, torch.float16, torch.float32)
_ACTS = {None: 0, "none": 0, "relu": 1, "silu": 2}


def group_norm_act_reference(x, num_groups, weight=None, bias=None, eps=1e-5, act=None, residual=None):
    """The definition in plain torch operations (fp32, or fp64 for fp64 inputs)."""
    n, c, h, w = x.shape
    xf = x if x.dtype == torch.float64 else x.float()
    g = xf.reshape(n, num_groups, c // num_groups * h * w)
    if g.numel():
        var, mean = torch.var_mean(g, dim=2, keepdim=True, unbiased=False)
        g = (g - mean) * torch.rsqrt(var + eps)
    z = g.reshape(n, c, h, w)
    if weight is not None:
        z = z * weight.to(z.dtype).view(1, c, 1, 1)
    if bias is not None:
        z = z + bias.to(z.dtype).view(1, c, 1, 1)
    if residual is not None:
        z = z + residual.to(z.dtype)
    if _ACTS[act] == 1:
        z = torch.relu(z)
    elif _ACTS[act] == 2:
        z = z * torch.sigmoid(z)
    return z.to(x.dtype)


def group_norm_act(x: torch.Tensor, num_groups: int, weight: Optional[torch.Tensor] = None,
                   bias: Optional[torch.Tensor] = None, eps: float = 1e-5, act: Optional[str] = None,
                   residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``act(GN(x) + residual)`` for a [N, C, H, W] map; ``act``: ``None`` / ``'none'``, ``'relu'`` or ``'silu'``.

    ``x`` and ``residual`` may be channels-last or channel slices of a channels-last buffer (other layouts are copied);
    the result is channels-last.  GPU types: bf16, fp16, fp32, statistics and gradients' sums in 32 and 64 bits;
    ``weight`` / ``bias``: [C] each, taken in fp32, either may be missing."""
    if x.dim() != 4:
        raise ValueError(f"group_norm_act: expected a [N, C, H, W] map, got {tuple(x.shape)}")
    c = x.shape[1]
    if act not in _ACTS:
        raise ValueError(f"group_norm_act: act must be None, 'none', 'relu' or 'silu', got {act!r}")
    if num_groups <= 0 or c == 0 or c % num_groups:
        raise ValueError(f"group_norm_act: {c} channels do not split into {num_groups} groups")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and (t.shape != (c,) or t.device != x.device):
            raise ValueError(f"group_norm_act: {name} must be [{c}] on {x.device}, got {tuple(t.shape)} on {t.device}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError(f"group_norm_act: residual {tuple(residual.shape)} {residual.dtype} {residual.device} does not "
                         f"match x {tuple(x.shape)} {x.dtype} {x.device}")
    if not B.use_hip(x):
        return group_norm_act_reference(x, num_groups, weight, bias, eps, act, residual)
    if x.dtype not in _TYPES:
        raise TypeError(f"group_norm_act: bf16, fp16 or fp32 maps, got {x.dtype}")
    if c > 0x7fffffff:
        raise NotImplementedError(f"group_norm_act: up to 2^31 - 1 channels, got {c}")
    return B.native().group_norm_act.default(x, weight, bias, residual, num_groups, eps, _ACTS[act])


class GroupNorm2d(nn.Module):
    """``nn.GroupNorm``-compatible parameters; forward takes ``BatchNorm2d``'s fusion flags, so that it stands where a
    ``BatchNorm2d`` does (``ops.conv_bn_act``): ``forward(x, relu, residual, dropout=p)`` is
    ``dropout(act(GN(x) + residual))``, dropout in training mode only."""

    batch_statistics = False       # nothing for a convolution's epilogue to collect, nothing to fold or to synchronise
    frozen = False

    def __init__(self, num_features: int, num_groups: int = 32, eps: float = 1e-5):
        super().__init__()
        if num_groups <= 0 or num_features % num_groups:
            raise ValueError(f"GroupNorm2d: {num_features} channels do not split into {num_groups} groups")
        self.num_features, self.num_groups, self.eps = num_features, num_groups, eps
        self.weight = nn.Parameter(torch.ones(num_features))
        self.bias = nn.Parameter(torch.zeros(num_features))

    def forward(self, x: torch.Tensor, relu: bool = False, residual: Optional[torch.Tensor] = None, stats=None,
                dropout: float = 0.0, out=None):
        """``stats`` and ``out`` (a convolution's sums, a concat slot) are ``BatchNorm2d``'s and have no use here: the
        result is an ordinary tensor, which ``ops.concat`` copies."""
        y = group_norm_act(x, self.num_groups, self.weight, self.bias, self.eps, "relu" if relu else None, residual)
        if dropout > 0.0 and self.training:
            from .dropout import dropout as _dropout
            y = _dropout(y, dropout)
        return y

    def extra_repr(self) -> str:
        return f"{self.num_features}, num_groups={self.num_groups}, eps={self.eps}"


def convert_group_norm(module: nn.Module, num_groups: int = 32) -> nn.Module:
    """``module`` with every ``BatchNorm2d`` replaced by a ``GroupNorm2d`` of the same weight and bias (in place; a module
    that is itself one is returned as its replacement), with the largest number of groups that divides both
    ``num_groups`` and its channels.  A module used in two places stays one module.  Layers that are stored wider than
    the architecture has them (Xception's 728-channel flow where it is padded) are refused, and nothing is replaced:
    a group's statistics would take in channels that do not exist."""
    if any(getattr(m, "stored_wider", False) for m in module.modules()):
        raise NotImplementedError("convert_group_norm: the module stores a BatchNorm2d wider than it is (Xception's 728 channels "
                                  "as 768, models.xception): zero channels would enter a group's statistics; DPAMD_X65_PAD=0 "
                                  "builds the model without them")
    return _convert(module, num_groups, {})


def _convert(module, num_groups, done):
    from .batchnorm import BatchNorm2d
    if module not in done:
        done[module] = module
        if isinstance(module, BatchNorm2d):
            gn = GroupNorm2d(module.num_features, math.gcd(num_groups, module.num_features), module.eps)
            gn.weight, gn.bias = module.weight, module.bias
            done[module] = gn.train(module.training)
        for name, child in module._modules.items():
            if child is not None:
                module._modules[name] = _convert(child, num_groups, done)
    return done[module]
