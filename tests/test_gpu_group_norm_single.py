"""Groups of one element: the normalised value is zero whatever the element, so is its gradient, exactly."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,c", [(1, 1), (3, 21), (2, 64), (5, 304), (9, 64), (1, 2048), (32, 728)])
@pytest.mark.parametrize("act,residual", [(None, False), (None, True), ("relu", False), ("relu", True), ("silu", True)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_a_group_of_one_element_has_no_gradient(n, c, act, residual, dtype):
    from distributedpytorch_amd import ops
    g = torch.Generator().manual_seed(n * c)
    x, r, dy = (torch.randn(n, c, 1, 1, generator=g).to(dtype).cuda() for _ in range(3))
    w, b = torch.randn(c, generator=g).cuda(), torch.randn(c, generator=g).cuda()
    leaves = [t.requires_grad_(True) for t in ((x, w, b, r) if residual else (x, w, b))]
    y = ops.group_norm_act(x, c, w, b, act=act, residual=r if residual else None)
    dx, dw, db, *dr = torch.autograd.grad(y, leaves, dy)
    assert not dx.any() and not dw.any()
    z = b.double().view(1, c, 1, 1).expand(n, c, 1, 1) + (r.double() if residual else 0.0)
    dz = {None: lambda: dy.double(), "relu": lambda: dy.double() * (z > 0),
          "silu": lambda: dy.double() * torch.sigmoid(z) * (1 + z * (1 - torch.sigmoid(z)))}[act]()
    # db: n terms in 32 bits; the native exponential of 16-bit types is a few 2^-23 off
    assert ((db.double() - dz.sum((0, 2, 3))).abs() <= (n + 64) * 2.0 ** -24 * dy.double().abs().sum((0, 2, 3)) + 1e-30).all()
    if residual:
        half = torch.finfo(dtype).eps / 2
        assert ((dr[0].double() - dz).abs() <= half * dz.abs() + 64 * 2.0 ** -24 * dy.double().abs() + 2.0 ** -25).all()
