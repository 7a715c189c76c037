"""Cross attention whose masks leave a few keys of a short sequence, or one key of a long one (csrc/cross_attention.hip).

Tolerances: those of tests/test_gpu_cross_attention.py."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from test_gpu_cross_attention import _check, _inputs  # noqa: E402
pytestmark = pytest.mark.gpu


def _gradients(q, k, v, dout, lens=None, mask=None):
    from distributedpytorch_amd import ops
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    return torch.autograd.grad(ops.cross_attention(*leaves, key_lengths=lens, key_mask=mask), leaves, dout)


def _keys(lk, *on):
    m = torch.zeros(lk, dtype=torch.bool)
    m[list(on)] = True
    return m


def _without(lk, *off):
    return ~_keys(lk, *off)


@pytest.mark.parametrize("mask", [
    _keys(40, 20, 35), _without(33, 0), _keys(33, 31, 32), _keys(33, 1, 2, 32), _keys(48, 15, 16, 40), _keys(63, 30, 62),
    _keys(64, 0, 63), _keys(64, 31, 32), _without(64, 32), _keys(63, 33, 34), _keys(40, 3, 4), _keys(17, 2, 16),
], ids=lambda m: f"{m.sum()} of {len(m)}")
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_key_that_takes_part_in_one_block_gets_its_gradient(mask, dtype):
    lk = len(mask)
    q, k, v, dout = _inputs(2, 3, lk, 4, 2, 64, dtype, seed=lk)
    mask = mask.expand(2, lk).cuda()
    _check(q, k, v, dout, mask=mask)
    dk, dv = _gradients(q, k, v, dout, mask=mask)[1:]
    assert (dk != 0).any(-1)[mask].all() and (dv != 0).any(-1)[mask].all()


@pytest.mark.parametrize("lk", [33, 40, 47, 63, 64, 100])
@pytest.mark.parametrize("density", [0.1, 0.5, 0.9])
@pytest.mark.parametrize("dim", [32, 64, 96, 128])
def test_random_masks_with_lengths_of_one_block(lk, density, dim):
    q, k, v, dout = _inputs(12, 3, lk, 2, 1, dim, torch.float16, seed=lk)
    g = torch.Generator().manual_seed(dim)
    mask = (torch.rand(12, lk, generator=g) < density).cuda()
    lens = torch.randint(0, min(lk, 64) + 1, (12,), generator=g).cuda()
    _check(q, k, v, dout, mask=mask)
    _check(q, k, v, dout, lens=lens, mask=mask)


@pytest.mark.parametrize("lq,lk,dim,at", [(50, 65, 64, (64, 0)), (1, 200, 128, (130, 199)), (33, 1023, 96, (1000, 3)),
                                          (3, 1100, 32, (1024, 1099)), (2, 20001, 64, (20000, 12345)), (600, 2049, 64, (2048, 700))])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_single_key_of_a_long_sequence_has_no_score_gradient(lq, lk, dim, at, dtype):
    """P = 1 whatever the score, however long the sequence is; image 2 has two keys, image 3 none."""
    q, k, v, dout = _inputs(4, lq, lk, 4, 2, dim, dtype, seed=lk)
    mask = torch.zeros(4, lk, dtype=torch.bool, device="cuda")
    for i, j in ((0, at[0]), (1, at[1]), (2, at[0]), (2, at[1])):
        mask[i, j] = True
    _check(q, k, v, dout, mask=mask)
    dq, dk, dv = _gradients(q, k, v, dout, mask=mask)
    for i in (0, 1, 3):
        assert not dq[i].any() and not dk[i].any()
    assert (dq[2] != 0).any(-1).all() and (dk[2] != 0).any(-1)[mask[2]].all() and (dv != 0).any(-1)[mask].all()
    # a length that leaves one of two unmasked keys
    lens = torch.full((4,), max(at), dtype=torch.int32, device="cuda")
    _check(q, k, v, dout, lens=lens, mask=mask)
    dq, dk, dv = _gradients(q, k, v, dout, lens=lens, mask=mask)
    assert not dq.any() and not dk.any() and (dv[2] != 0).any(-1).sum() == dv.shape[2]


@pytest.mark.parametrize("lk,kind", [(1, "one key"), (60, "mask"), (60, "length"), (200, "mask"), (200, "length"), (5000, "mask")])
def test_a_nan_query_reaches_the_gradients_of_a_single_key(lk, kind):
    """P of that row is NaN, as its output is; the other rows' dq are zeros."""
    from distributedpytorch_amd import ops
    q, k, v, dout = _inputs(2, 40, lk, 4, 2, 64, torch.bfloat16, seed=lk)
    q[0, 7, 3, 5] = float("nan")
    lens = torch.ones(2, dtype=torch.int32, device="cuda") if kind == "length" else None
    at = lk - 1 if kind == "mask" else 0
    mask = _keys(lk, at).expand(2, lk).cuda() if kind == "mask" else None
    out = ops.cross_attention(q, k, v, key_lengths=lens, key_mask=mask)
    dq, dk, dv = _gradients(q, k, v, dout, lens, mask)
    assert out[0, 7, 3].isnan().all() and dq[0, 7, 3].isnan().all()
    assert dk[0, at, 1].isnan().all() and dv[0, at, 1].isnan().all()
    for t, where in ((out, (0, 7, 3)), (dq, (0, 7, 3)), (dk, (0, at, 1)), (dv, (0, at, 1))):
        t[where] = 0
        assert not t.isnan().any()
    assert not dq.any() and not dk.any()
