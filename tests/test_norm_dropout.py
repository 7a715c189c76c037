"""Group norm with an activation and seeded dropout on the CPU path: the definitions, and what the entry points refuse."""
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from distributedpytorch_amd import ops  # noqa: E402
from distributedpytorch_amd.ops.dropout import dropout_keep, dropout_threshold  # noqa: E402


@pytest.mark.parametrize("c,groups", [(8, 2), (21, 7), (6, 6), (5, 1)])
@pytest.mark.parametrize("act", [None, "relu", "silu"])
def test_group_norm_matches_the_definition_in_numpy(c, groups, act):
    g = torch.Generator().manual_seed(c * 10 + groups)
    x = torch.randn(2, c, 3, 5, generator=g, dtype=torch.float64)
    w, b = torch.randn(c, generator=g, dtype=torch.float64), torch.randn(c, generator=g, dtype=torch.float64)
    r = torch.randn(2, c, 3, 5, generator=g, dtype=torch.float64)
    y = ops.group_norm_act(x, groups, w, b, 1e-5, act=act, residual=r).numpy()
    xs = x.numpy().reshape(2, groups, -1)
    xh = (xs - xs.mean(2, keepdims=True)) / np.sqrt(xs.var(2, keepdims=True) + 1e-5)
    z = xh.reshape(2, c, 3, 5) * w.numpy()[:, None, None] + b.numpy()[:, None, None] + r.numpy()
    want = {None: z, "relu": np.maximum(z, 0), "silu": z / (1 + np.exp(-z))}[act]
    np.testing.assert_allclose(y, want, rtol=1e-12, atol=1e-12)


def test_group_norm_gradient_against_differences():
    g = torch.Generator().manual_seed(1)
    mk = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64, requires_grad=True)  # noqa: E731
    args = (mk(2, 6, 2, 3), mk(6), mk(6), mk(2, 6, 2, 3))
    assert torch.autograd.gradcheck(
        lambda x, w, b, r: ops.group_norm_act(x, 3, w, b, 1e-5, act="silu", residual=r), args)


def test_group_norm_of_nothing():
    x = torch.zeros(0, 8, 4, 4)
    assert ops.group_norm_act(x, 2).shape == (0, 8, 4, 4)
    assert ops.group_norm_act(torch.zeros(2, 8, 0, 4), 2, act="relu").shape == (2, 8, 0, 4)


@pytest.mark.parametrize("kw,err", [
    (dict(x=torch.zeros(2, 8, 4)), ValueError), (dict(num_groups=3), ValueError), (dict(num_groups=0), ValueError),
    (dict(act="tanh"), ValueError), (dict(weight=torch.ones(4)), ValueError), (dict(bias=torch.ones(9)), ValueError),
    (dict(residual=torch.zeros(2, 8, 4, 3)), ValueError),
    (dict(residual=torch.zeros(2, 8, 4, 4, dtype=torch.bfloat16)), ValueError),
])
def test_group_norm_refusals(kw, err):
    args = dict(x=torch.zeros(2, 8, 4, 4), num_groups=2)
    args.update(kw)
    with pytest.raises(err):
        ops.group_norm_act(**args)


def _philox(counter, key):
    """Philox4x32-10 with Python's integers."""
    c, k = list(counter), list(key)
    for _ in range(10):
        p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(p1 >> 32) ^ c[1] ^ k[0], p1 & 0xFFFFFFFF, (p0 >> 32) ^ c[3] ^ k[1], p0 & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def test_philox_known_answers():
    # the published known-answer vectors of philox4x32-10
    assert _philox((0, 0, 0, 0), (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert _philox((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


@pytest.mark.parametrize("seed", [0, 1, 0x123456789ABCDEF0, 0xFFFFFFFFFFFFFFFF])
@pytest.mark.parametrize("p", [0.1, 0.5, 1e-9])
def test_dropout_keep_is_philox(seed, p):
    keep = dropout_keep(43, seed, p).tolist()
    want = []
    for j in range(6):
        for word in _philox((j, 0, 0, 0), (seed & 0xFFFFFFFF, seed >> 32)):
            want += [(word & 0xFFFF) >= dropout_threshold(p), (word >> 16) >= dropout_threshold(p)]
    assert keep == want[:43]
    signed = seed - (1 << 64) if seed >> 63 else seed
    assert torch.equal(dropout_keep(43, torch.tensor([signed]), p), torch.tensor(keep))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
@pytest.mark.parametrize("layout", ["contiguous", "channels_last", "sliced"])
def test_dropout_values_and_gradients(dtype, layout):
    x = torch.randn(2, 5, 3, 7, dtype=dtype)
    if layout == "channels_last":
        x = x.contiguous(memory_format=torch.channels_last)
    elif layout == "sliced":
        x = torch.randn(2, 5, 3, 9, dtype=dtype)[..., 1:8]
    r = torch.randn(2, 5, 3, 7, dtype=dtype)
    x, r = x.detach().requires_grad_(True), r.requires_grad_(True)
    y = ops.dropout(x, 0.3, seed=77, residual=r)
    thr = dropout_threshold(0.3)
    keep = dropout_keep(x.numel(), 77, 0.3)
    keep = keep.view(2, 3, 7, 5).permute(0, 3, 1, 2) if layout == "channels_last" else keep.view(2, 5, 3, 7)
    wide = dtype if dtype == torch.float64 else torch.float32
    s = 65536.0 / (65536.0 - thr)
    assert torch.equal(y, (torch.where(keep, x.to(wide) * s, torch.zeros((), dtype=wide)) + r.to(wide)).to(dtype))
    dy = torch.randn(2, 5, 3, 7).to(dtype)
    dx, dr = torch.autograd.grad(y, (x, r), dy)
    assert torch.equal(dx, torch.where(keep, dy.to(wide) * s, torch.zeros((), dtype=wide)).to(dtype))
    assert torch.equal(dr, dy)


def test_dropout_ends_of_the_range():
    x = torch.tensor([1.0, float("inf"), float("nan")])
    r = torch.ones(3)
    assert ops.dropout(x[:1], 0.0) is not None and torch.equal(ops.dropout(r, 0.0, residual=r), r + r)
    assert torch.equal(ops.dropout(x, 1.0, seed=3), torch.zeros(3))           # dropped elements are zeros, whatever they held
    assert torch.equal(ops.dropout(x, 1.0, seed=3, residual=r), r)
    assert torch.equal(ops.dropout(r, 0.5, training=False), r)
    assert ops.dropout(torch.zeros(0, 3), 0.5, seed=1).shape == (0, 3)


def test_dropout_draws_a_new_mask_each_call():
    x = torch.ones(4096)
    a, b = ops.dropout(x, 0.5), ops.dropout(x, 0.5)
    assert not torch.equal(a, b)
    # kept: binomial(4096, 1/2), standard deviation 32: seven of them
    assert abs(int((a != 0).sum()) - 2048) < 7 * 32


@pytest.mark.parametrize("kw,err", [
    (dict(p=-0.1), ValueError), (dict(p=1.5), ValueError), (dict(p=float("nan")), ValueError),
    (dict(residual=torch.zeros(3)), ValueError), (dict(residual=torch.zeros(4, dtype=torch.float64)), ValueError),
    (dict(seed=torch.zeros(2, dtype=torch.int64)), ValueError), (dict(seed=torch.zeros(1)), ValueError),
    (dict(seed=1.5), TypeError), (dict(x=torch.zeros(4, dtype=torch.int32)), TypeError),
])
def test_dropout_refusals(kw, err):
    args = dict(x=torch.zeros(4), p=0.5)
    args.update(kw)
    with pytest.raises(err):
        ops.dropout(**args)
