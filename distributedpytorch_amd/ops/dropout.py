"""Dropout whose mask is a function of (seed, position) and is never stored (csrc/dropout.hip, csrc/autograd.cpp).

The keep decision of an element comes from Philox4x32-10 (Salmon et al. 2011) under a 64-bit seed: block ``j`` of eight
elements in memory order has the counter ``(j, j >> 32, 0, 0)``, each 32-bit word decides two elements, and backward
computes the same decisions again.  CPU tensors / ``set_backend('torch')`` run the same generator in plain torch
operations: one seed gives one mask everywhere.
"""
from __future__ import annotations

import operator
from typing import Optional, Union

import torch

from . import _backend as B

_TYPES = (torch.bfloat16, torch.float16, torch.float32)
_LOW = 0xFFFFFFFF


def dropout_threshold(p: float) -> int:
    """``p`` in steps of 1/65536: an element is dropped where 16 random bits are below it (1 and 65535 are the ends of
    0 < p < 1; ``p = 1`` drops everything)."""
    return 65536 if p >= 1.0 else min(65535, max(1, int(round(p * 65536))))


def dropout_keep(count: int, seed, p: float, device=None) -> torch.Tensor:
    """bool [count]: the keep decisions of ``count`` elements, in plain torch operations (``seed``: int or int64 tensor)."""
    block = torch.arange((count + 7) // 8, dtype=torch.int64, device=device)
    a, b = block & _LOW, block >> 32
    c, d = torch.zeros_like(block), torch.zeros_like(block)
    k0, k1 = seed & _LOW, (seed >> 32) & _LOW
    for _ in range(10):
        # (64-bit products wrap; their low and high words are those of the unsigned ones)
        lo, hi = a * 0xD2511F53, c * 0xCD9E8D57
        a, b, c, d = ((hi >> 32) & _LOW) ^ b ^ k0, hi & _LOW, ((lo >> 32) & _LOW) ^ d ^ k1, lo & _LOW
        k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
    words = torch.stack((a, b, c, d), dim=1)
    return torch.stack((words & 0xFFFF, words >> 16), dim=2).reshape(-1)[:count] >= dropout_threshold(p)


def _dense(t: torch.Tensor) -> torch.Tensor:
    """``t`` itself where its elements fill their memory without gaps in one of torch's two layouts, else a copy."""
    if t.is_contiguous() or (t.dim() == 4 and t.is_contiguous(memory_format=torch.channels_last)):
        return t
    return t.contiguous()


def _like(t: torch.Tensor, ref: torch.Tensor) -> torch.Tensor:
    """``t`` in the memory order of the dense tensor ``ref``."""
    if t.stride() == ref.stride():
        return t
    out = torch.empty_like(ref, dtype=t.dtype)
    return out.copy_(t)


def _memory_order(t: torch.Tensor) -> torch.Tensor:
    """The elements of a dense tensor as a flat view, in memory order."""
    return t.as_strided((t.numel(),), (1,))


def _run(x, residual, p, seed):
    """``x`` dense; ``residual`` in the same order or None."""
    keep = dropout_keep(x.numel(), seed, p, x.device)
    wide = x if x.dtype == torch.float64 else x.float()
    thr = dropout_threshold(p)
    flat = torch.where(keep, _memory_order(wide) * (65536.0 / (65536.0 - thr) if thr < 65536 else 0.0),
                       torch.zeros((), dtype=wide.dtype, device=x.device))
    if residual is not None:
        flat = flat + _memory_order(residual).to(flat.dtype)
    out = torch.empty_like(x)
    _memory_order(out).copy_(flat)
    return out


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed):
        x = _dense(x)
        ctx.p, ctx.seed, ctx.strides = p, None if isinstance(seed, torch.Tensor) else seed, x.stride()
        ctx.save_for_backward(seed if isinstance(seed, torch.Tensor) else None)
        return _run(x, None if residual is None else _like(residual, x), p, seed)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        (held,) = ctx.saved_tensors
        dx = None
        if ctx.needs_input_grad[0]:
            g = dy
            if g.stride() != ctx.strides:          # the mask follows the memory order of the forward's input
                g = torch.empty_strided(dy.shape, ctx.strides, dtype=dy.dtype, device=dy.device).copy_(dy)
            dx = _run(g, None, ctx.p, held if held is not None else ctx.seed)
        return dx, dy if ctx.needs_input_grad[1] else None, None, None


def dropout(x: torch.Tensor, p: float = 0.5, training: bool = True, seed: Optional[Union[int, torch.Tensor]] = None,
            residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``dropout(x) (+ residual)`` in one pass; the mask is recomputed in backward instead of being kept.

    ``p``: probability of dropping an element, in steps of 1/65536.  ``seed``: ``None`` draws one per call from torch's
    seed, the rank and a call counter (captured training steps mix their step number in, ``TrainEngine.graph_step``); an
    ``int`` is used as it is (its low 64 bits); an int64 tensor of one element on ``x``'s device is read when the kernel
    runs, so a captured graph draws a new mask when the program has written a new seed between replays — it must hold
    the same value when backward runs.  ``x`` may be contiguous or channels-last (the mask follows memory order); other
    layouts are copied.  A call that is run again for its backward pass (activation checkpointing) needs a ``seed`` of its
    own: a drawn one would be another.  GPU types: bf16, fp16, fp32."""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout: p must lie in [0, 1], got {p}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError(f"dropout: residual {tuple(residual.shape)} {residual.dtype} {residual.device} does not match "
                         f"x {tuple(x.shape)} {x.dtype} {x.device}")
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1 or seed.device != x.device:
            raise ValueError("dropout: a seed tensor holds one int64 on x's device, got "
                             f"{tuple(seed.shape)} {seed.dtype} {seed.device}")
        seed = seed.reshape(1)
    if not training or p == 0.0:
        return x if residual is None else x + residual
    if not x.is_floating_point() or (B.use_hip(x) and x.dtype not in _TYPES):
        raise TypeError(f"dropout: bf16, fp16 or fp32 tensors, got {x.dtype}")
    use_word = seed is None
    if use_word:
        from .batchnorm import _dropout_key
        seed = _dropout_key(p)[1]
    elif not isinstance(seed, torch.Tensor):
        seed = operator.index(seed) & 0xFFFFFFFFFFFFFFFF
    if B.use_hip(x):
        held = isinstance(seed, torch.Tensor)
        number = 0 if held else seed - (1 << 64) if seed >= 1 << 63 else seed            # (as a signed 64-bit number)
        return B.native().dropout.default(x, residual, dropout_threshold(p), number, seed if held else None, use_word)
    if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)):
        return _Dropout.apply(x, residual, p, seed)
    x = _dense(x)
    return _run(x, None if residual is None else _like(residual, x), p, seed)
