"""Attention of one sequence's queries over another's keys and values (csrc/cross_attention.hip,
csrc/autograd.cpp).

``position_attention`` (ops.attention) is DANet's: one head, every position of a map over the same map, no mask.  Here the
two lengths differ, heads are split and may share keys, and images may hold fewer keys than the tensor has room for — a
decoder's positions over an encoder's, or a single query over a whole map.  CPU tensors / ``set_backend('torch')`` run
plain torch operations.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _backend as B

_TYPES = (torch.bfloat16, torch.float16)
MAX_DIM = 128
MAX_LENGTH = 1 << 29


def cross_attention_reference(q, k, v, key_lengths=None, key_mask=None, scale=None):
    """The definition in plain torch operations (fp32, or fp64 for fp64 inputs)."""
    b, lq, hq, d = q.shape
    lk, hk = k.shape[1], k.shape[2]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    wide = torch.float64 if q.dtype == torch.float64 else torch.float32
    on = torch.ones((b, lk), dtype=torch.bool, device=q.device)
    if key_lengths is not None:
        on = on & (torch.arange(lk, device=q.device) < key_lengths[:, None])
    if key_mask is not None:
        on = on & key_mask
    zero = torch.zeros((), dtype=wide, device=q.device)
    kf, vf = (torch.where(on[:, :, None, None], t.to(wide), zero).repeat_interleave(hq // hk, dim=2).permute(0, 2, 1, 3)
              for t in (k, v))
    s = torch.matmul(q.to(wide).permute(0, 2, 1, 3), kf.transpose(2, 3).contiguous()) * scale
    some = on.any(dim=1)[:, None, None, None]
    s = torch.where(on[:, None, None, :], s, torch.full((), -math.inf, dtype=wide, device=q.device))
    p = torch.softmax(torch.where(some, s, zero), dim=-1) if lk else s
    o = torch.matmul(torch.where(some, p, zero), vf.contiguous())
    return o.permute(0, 2, 1, 3).contiguous().to(q.dtype)


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, key_lengths: Optional[torch.Tensor] = None,
                    key_mask: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """``softmax(scale · q kᵀ) v`` per head: ``q`` [B, Lq, Hq, D], ``k`` and ``v`` [B, Lk, Hk, D] -> [B, Lq, Hq, D].

    ``Hq`` is a multiple of ``Hk``: neighbouring query heads share a key / value head.  ``key_lengths``: int tensor [B],
    image ``i`` has its first ``key_lengths[i]`` keys (values outside [0, Lk] count as the nearer end); ``key_mask``:
    bool [B, Lk], True where a key takes part.  Keys that take no part may hold anything; a row without a key gives
    zeros and zero gradients.  ``scale``: positive, default ``1 / sqrt(D)``.  A channels-last map [N, C, H, W] is the
    sequence ``map.permute(0, 2, 3, 1).reshape(N, H * W, heads, C // heads)`` (a view).
    GPU types: bf16, fp16; head widths up to 128.  Scores, sums and statistics are held in 32 bits; probabilities, and the
    gradients of scores, are rounded to the tensors' type before the product they enter."""
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape:
        raise ValueError("cross_attention: q [B, Lq, Hq, D], k and v [B, Lk, Hk, D], got "
                         f"{tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    b, lq, hq, d = q.shape
    lk, hk = k.shape[1], k.shape[2]
    if k.shape[0] != b or k.shape[3] != d or d == 0 or hk == 0 or hq == 0 or hq % hk:
        raise ValueError(f"cross_attention: q {tuple(q.shape)} and k {tuple(k.shape)} differ in images or head width, or "
                         f"{hq} query heads do not share {hk} key heads evenly")
    if k.dtype != q.dtype or v.dtype != q.dtype or k.device != q.device or v.device != q.device:
        raise ValueError("cross_attention: q, k and v must have one type and one device")
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    if not 0.0 < scale < math.inf:
        raise ValueError(f"cross_attention: scale must be positive and finite, got {scale}")
    if key_lengths is not None:
        if key_lengths.shape != (b,) or key_lengths.dtype not in (torch.int32, torch.int64) or key_lengths.device != q.device:
            raise ValueError(f"cross_attention: key_lengths must be int32 or int64 [{b}] on {q.device}, got "
                             f"{tuple(key_lengths.shape)} {key_lengths.dtype} on {key_lengths.device}")
    if key_mask is not None:
        if key_mask.shape != (b, lk) or key_mask.dtype != torch.bool or key_mask.device != q.device:
            raise ValueError(f"cross_attention: key_mask must be bool [{b}, {lk}] on {q.device}, got "
                             f"{tuple(key_mask.shape)} {key_mask.dtype} on {key_mask.device}")
    if not B.use_hip(q):
        return cross_attention_reference(q, k, v, key_lengths, key_mask, scale)
    if q.dtype not in _TYPES:
        raise TypeError(f"cross_attention kernels: bf16 or fp16, got {q.dtype}; set_backend('torch') runs the plain formulation")
    if d > MAX_DIM:
        raise NotImplementedError(f"cross_attention kernels: head widths up to {MAX_DIM}, got {d}; set_backend('torch') "
                                  "runs the plain formulation")
    if max(b, lq * (hq // hk), lk, hq) > MAX_LENGTH:
        raise NotImplementedError(f"cross_attention kernels: up to {MAX_LENGTH} images, heads, keys, and positions times the "
                                  f"query heads of a key head, got q {tuple(q.shape)}, k {tuple(k.shape)}")
    if q.numel() == 0 or lk == 0:
        return (q * 0).nan_to_num(0.0) + (k.sum() + v.sum()) * 0      # zeros, tied to all three inputs
    lens = key_lengths                               # (the kernels limit the values to [0, Lk])
    if lens is not None:
        lens = (lens if lens.dtype == torch.int32 else lens.clamp(0, lk).to(torch.int32)).contiguous()
    mask = None if key_mask is None else (key_mask if key_mask.stride(1) == 1 or lk == 1 else key_mask.contiguous())
    if d % 8:
        # zero columns are exact: they add nothing to q kᵀ, and zero value columns are sliced off again
        q, k, v = (torch.nn.functional.pad(t, (0, 8 - d % 8)) for t in (q, k, v))
    out = B.native().cross_attention.default(q, k, v, lens, mask, scale)
    return out[..., :d] if d % 8 else out
