"""Group normalisation of channels-last maps fused with a residual and an activation (csrc/group_norm.hip).

The counterpart of ``batch_norm_act`` whose statistics come from one image's group of channels: nothing depends on the
batch, so it serves training at a few images per GPU, and evaluation computes what training computes.  CPU tensors /
``set_backend('torch')`` run plain torch operations.
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import Optional

import torch
import torch.nn as nn

from . import _backend as B
from .concat import row_stride

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_ACTS = {None: 0, "none": 0, "relu": 1, "silu": 2}
_sigs = False


def _lib():
    global _sigs
    lib = B.lib()
    if not _sigs:
        V, L, I, F = ctypes.c_void_p, ctypes.c_long, ctypes.c_int, ctypes.c_float
        lib.dp_gn_workspace.argtypes = [L, L, I, I, I]
        lib.dp_gn_workspace.restype = L
        lib.dp_gn_fwd.argtypes = [V] * 7 + [L, L, I, I, L, L, F, I, I, V]
        lib.dp_gn_bwd.argtypes = [V] * 11 + [L, L, I, I, L, L, L, I, I, V]
        _sigs = True
    return lib


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


def _rows(t: torch.Tensor):
    """(tensor, elements between rows): ``t`` as it is when its memory is NHWC rows (a channels-last map or a channel
    slice of one), a channels-last copy otherwise."""
    ld = t.shape[1]
    if t.is_contiguous(memory_format=torch.channels_last):
        return t, ld
    ld = row_stride(t)
    if ld is None:
        t = t.contiguous(memory_format=torch.channels_last)
        ld = t.shape[1]
    return t, ld


def _p(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _vec(t: Optional[torch.Tensor]):
    if t is None:
        return None
    t = t.detach()
    return t if t.dtype == torch.float32 and t.is_contiguous() else t.float().contiguous()


def _new(x: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(x, memory_format=torch.channels_last)


@functools.lru_cache(maxsize=4096)
def _workspace_floats(n, hw, c, groups, esize) -> int:
    return int(_lib().dp_gn_workspace(n, hw, c, groups, esize))


def _workspace(x, n, hw, c, groups):
    return torch.empty(_workspace_floats(n, hw, c, groups, x.element_size()), dtype=torch.float32, device=x.device)


def _forward(x, groups, weight, bias, eps, act, residual):
    n, c, h, w = x.shape
    y = _new(x)
    stats = torch.empty((n, groups, 2), dtype=torch.float64, device=x.device)
    if x.numel():
        x, ldx = _rows(x)
        ldr = c
        if residual is not None:
            residual, ldr = _rows(residual)
        ws = _workspace(x, n, h * w, c, groups)
        B.launch("gn_fwd", _lib().dp_gn_fwd, x, _p(x), _p(residual), _p(weight), _p(bias), _p(y), _p(stats), _p(ws), n, h * w,
                 c, groups, ldx, ldr, eps, act, _DTYPES[x.dtype])
    return y, stats


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, groups, eps, act):
        w32, b32 = _vec(weight), _vec(bias)
        y, stats = _forward(x, groups, w32, b32, eps, act, residual)
        # an activation's derivative needs z: the residual is kept for it (without one its gradient is dy itself)
        ctx.save_for_backward(x, residual if act else None, w32, b32, stats)
        ctx.meta = (groups, act, None if weight is None else weight.dtype, None if bias is None else bias.dtype)
        return y

    @staticmethod
    def backward(ctx, dy):
        B.first_order("group_norm_act")
        x, residual, w32, b32, stats = ctx.saved_tensors
        groups, act, wdtype, bdtype = ctx.meta
        n, c, h, w = x.shape
        dx = _new(x)
        dres = _new(x) if residual is not None else None
        dw = None if wdtype is None else torch.empty_like(w32)
        db = None if bdtype is None else torch.empty_like(b32)
        if x.numel():
            x, ldx = _rows(x)
            g, ldd = _rows(dy)
            ldr = c
            if residual is not None:
                residual, ldr = _rows(residual)
            ws = _workspace(x, n, h * w, c, groups)
            B.launch("gn_bwd", _lib().dp_gn_bwd, x, _p(g), _p(x), _p(residual), _p(w32), _p(b32), _p(stats), _p(dx), _p(dres),
                     _p(dw), _p(db), _p(ws), n, h * w, c, groups, ldx, ldr, ldd, act, _DTYPES[x.dtype])
        else:
            for t in (dw, db):
                if t is not None:
                    t.zero_()
        if dres is None and ctx.needs_input_grad[3]:
            dres = dy                                     # no activation: the residual's gradient is dy
        if dw is not None and wdtype != torch.float32:
            dw = dw.to(wdtype)
        if db is not None and bdtype != torch.float32:
            db = db.to(bdtype)
        return dx, dw, db, dres, None, None, None


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
    if x.dtype not in _DTYPES:
        raise TypeError(f"group_norm_act: bf16, fp16 or fp32 maps, got {x.dtype}")
    if c > 0x7fffffff:
        raise NotImplementedError(f"group_norm_act: up to 2^31 - 1 channels, got {c}")
    code = _ACTS[act]
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual)):
        return _GroupNormAct.apply(x, weight, bias, residual, num_groups, eps, code)
    return _forward(x, num_groups, _vec(weight), _vec(bias), eps, code, residual)[0]


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
    ``num_groups`` and its channels.  A module used in two places stays one module."""
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
