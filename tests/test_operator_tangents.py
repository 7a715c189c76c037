"""Forward-mode derivatives: the plain formulations carry a tangent, the C++ operators refuse one instead of dropping it."""
import os
import sys

import pytest
import torch
from torch.autograd import forward_ad

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from distributedpytorch_amd import ops  # noqa: E402
from distributedpytorch_amd.ops import _backend as B  # noqa: E402


def _inputs(device):
    torch.manual_seed(0)
    mk = lambda *s, t=torch.float32: torch.randn(*s, device=device).to(t)  # noqa: E731
    bf = torch.bfloat16
    return {"norm": dict(x=mk(1, 8, 4, 4), weight=mk(8), bias=mk(8), residual=mk(1, 8, 4, 4)),
            "dropout": dict(x=mk(1, 8, 4, 4), residual=mk(1, 8, 4, 4)),
            "attention": dict(q=mk(1, 3, 2, 8, t=bf), k=mk(1, 5, 2, 8, t=bf), v=mk(1, 5, 2, 8, t=bf))}


NAMES = [("norm", n) for n in ("x", "weight", "bias", "residual")] + [("dropout", n) for n in ("x", "residual")] + \
    [("attention", n) for n in ("q", "k", "v")]


def _dual(inputs, name, wanted):
    return {n: forward_ad.make_dual(t.requires_grad_(wanted), torch.ones_like(t)) if n == name else t for n, t in inputs.items()}


@pytest.mark.parametrize("wanted", [False, True])
@pytest.mark.parametrize("op,name", NAMES)
def test_native_operators_refuse_a_tangent(op, name, wanted):
    native = B.native()
    call = {"norm": lambda x, weight, bias, residual: native.group_norm_act.default(x, weight, bias, residual, 2, 1e-5, 1),
            "dropout": lambda x, residual: native.dropout.default(x, residual, 1000, 1, None, False),
            "attention": lambda q, k, v: native.cross_attention.default(q, k, v, None, None, 1.0)}[op]
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(**_dual(_inputs("cpu")[op], name, wanted))


def _public(op):
    return {"norm": lambda x, weight, bias, residual: ops.group_norm_act(x, 2, weight, bias, act="relu", residual=residual),
            "dropout": lambda x, residual: ops.dropout(x, 0.25, seed=3, residual=residual), "attention": ops.cross_attention}[op]


@pytest.mark.parametrize("op,name", NAMES)
def test_plain_formulations_carry_a_tangent(op, name):
    inputs = {n: t.double() for n, t in _inputs("cpu")[op].items()}
    with forward_ad.dual_level():
        tangent = forward_ad.unpack_dual(_public(op)(**_dual(inputs, name, False))).tangent
    assert tangent is not None
    step = 1e-6
    up, down = ({n: t + (s * step if n == name else 0.0) for n, t in inputs.items()} for s in (1, -1))
    want = (_public(op)(**up) - _public(op)(**down)) / (2 * step)
    assert (tangent - want).abs().max() < 1e-6 * (1 + want.abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("op,name", NAMES)
def test_public_functions_refuse_a_tangent_on_the_gpu(op, name):
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            _public(op)(**_dual(_inputs("cuda")[op], name, False))
    with forward_ad.dual_level():                          # a level without tangents changes nothing
        out = _public(op)(**_inputs("cuda")[op])
    assert torch.isfinite(out).all()
