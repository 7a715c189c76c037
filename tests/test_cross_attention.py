"""Cross attention on the CPU path: the definition, rows without keys, and what the entry point refuses."""
import math
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from distributedpytorch_amd import ops  # noqa: E402


def _loop(q, k, v, on, scale):
    """Row by row in numpy, over the keys that take part."""
    b, lq, hq, d = q.shape
    hk = k.shape[2]
    out = np.zeros((b, lq, hq, d))
    for i in range(b):
        keys = np.nonzero(on[i])[0]
        if len(keys) == 0:
            continue
        for j in range(hq):
            kk, vv = k[i, keys, j // (hq // hk)], v[i, keys, j // (hq // hk)]
            for r in range(lq):
                s = kk @ q[i, r, j] * scale
                e = np.exp(s - s.max())
                out[i, r, j] = e / e.sum() @ vv
    return out


@pytest.mark.parametrize("lq,lk,hq,hk,d", [(1, 1, 1, 1, 1), (3, 7, 4, 2, 5), (5, 2, 3, 3, 8), (2, 9, 6, 1, 4)])
@pytest.mark.parametrize("masks", ["none", "lengths", "both"])
def test_cross_attention_matches_a_loop(lq, lk, hq, hk, d, masks):
    g = torch.Generator().manual_seed(lq * 100 + lk)
    q, k, v = (torch.randn(3, n, h, d, generator=g, dtype=torch.float64) for n, h in ((lq, hq), (lk, hk), (lk, hk)))
    on = np.ones((3, lk), dtype=bool)
    lens = mask = None
    if masks != "none":
        lens = torch.tensor([lk, 0, max(1, lk - 1)])
        on &= np.arange(lk)[None] < lens.numpy()[:, None]
    if masks == "both":
        mask = torch.rand(3, lk, generator=g) < 0.6
        on &= mask.numpy()
        k[~mask], v[~mask] = float("nan"), float("inf")
    got = ops.cross_attention(q, k, v, key_lengths=lens, key_mask=mask, scale=0.7)
    want = _loop(q.numpy(), k.numpy(), v.numpy(), on, 0.7)
    np.testing.assert_allclose(got.numpy(), want, rtol=1e-12, atol=1e-13)


def test_cross_attention_gradient_against_differences():
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(2, n, h, 3, generator=g, dtype=torch.float64, requires_grad=True)
               for n, h in ((2, 4), (5, 2), (5, 2)))
    mask = torch.tensor([[1, 0, 1, 1, 0], [0, 0, 0, 0, 0]], dtype=torch.bool)
    assert torch.autograd.gradcheck(lambda a, b, c: ops.cross_attention(a, b, c, key_mask=mask), (q, k, v))
    assert torch.autograd.gradcheck(lambda a, b, c: ops.cross_attention(a, b, c, key_lengths=torch.tensor([5, 2])), (q, k, v))


def test_cross_attention_empty_sizes():
    q, k = torch.randn(2, 3, 4, 8, requires_grad=True), torch.randn(2, 0, 2, 8, requires_grad=True)
    out = ops.cross_attention(q, k, k)
    assert torch.equal(out, torch.zeros_like(q))
    out.sum().backward()
    assert torch.equal(q.grad, torch.zeros_like(q)) and k.grad.shape == k.shape
    assert ops.cross_attention(q[:, :0], torch.randn(2, 5, 2, 8), torch.randn(2, 5, 2, 8)).shape == (2, 0, 4, 8)


def test_cross_attention_default_scale():
    q, k, v = torch.randn(1, 2, 1, 16), torch.randn(1, 3, 1, 16), torch.randn(1, 3, 1, 16)
    assert torch.equal(ops.cross_attention(q, k, v), ops.cross_attention(q, k, v, scale=1 / math.sqrt(16)))


@pytest.mark.parametrize("kw", [
    dict(q=torch.zeros(2, 3, 8)), dict(q=torch.zeros(3, 3, 4, 8)), dict(q=torch.zeros(2, 3, 4, 16)),
    dict(q=torch.zeros(2, 3, 3, 8)), dict(v=torch.zeros(2, 6, 2, 8)), dict(v=torch.zeros(2, 5, 2, 8, dtype=torch.float64)),
    dict(q=torch.zeros(2, 3, 4, 8, dtype=torch.bfloat16)), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
    dict(scale=float("inf")), dict(key_lengths=torch.zeros(3, dtype=torch.int32)), dict(key_lengths=torch.zeros(2)),
    dict(key_mask=torch.ones(2, 4, dtype=torch.bool)), dict(key_mask=torch.ones(2, 5)),
    dict(key_mask=torch.ones(2, 1, 5, dtype=torch.bool)),
])
def test_cross_attention_refusals(kw):
    args = dict(q=torch.zeros(2, 3, 4, 8), k=torch.zeros(2, 5, 2, 8), v=torch.zeros(2, 5, 2, 8))
    args.update(kw)
    with pytest.raises(ValueError):
        ops.cross_attention(**args)
