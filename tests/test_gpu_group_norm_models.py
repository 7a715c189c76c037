"""Group norm inside models on the GPU: Xception's separable units, and FCN and DANet."""
import copy
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
pytestmark = pytest.mark.gpu

from distributedpytorch_amd import ops  # noqa: E402

HALF = 2.0 ** -8                                       # a rounding to bf16, relative


def _rel(got, want):
    return float((got.detach().double().cpu() - want.detach().double()).norm() / want.detach().double().norm())


def _weights(module, seed):
    """Norms with weights and shifts of their own; every convolution's gain near 1."""
    g = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for m in module.modules():
            if isinstance(m, (ops.BatchNorm2d, ops.GroupNorm2d)):
                m.weight.copy_(1 + 0.2 * torch.randn(m.weight.shape, generator=g))
                m.bias.copy_(0.2 * torch.randn(m.bias.shape, generator=g))
    return module


def _convert(module, which):
    for m in list(module.modules()):
        for name, child in m.named_children():
            if isinstance(child, ops.BatchNorm2d) and which(m, name):
                setattr(m, name, ops.convert_group_norm(child))
    return module


PLACES = {"all": lambda m, name: True, "behind the depthwise": lambda m, name: hasattr(m, "pointwise"),
          "behind the pointwise": lambda m, name: not hasattr(m, "pointwise")}


@pytest.mark.parametrize("training", [True, False])
@pytest.mark.parametrize("place", list(PLACES))
@pytest.mark.parametrize("cin,cout,stride", [(64, 128, 2), (128, 128, 1)])
def test_xception_block_with_group_norm_matches_fp32(cin, cout, stride, place, training):
    """Against the same block in fp32 on the CPU.  Three units of two convolutions and two norms, and the shortcut: 16 maps
    and 8 weights on the way are rounded once to bf16; as many again, and as many gradients, on the way back.  Sixteen
    roundings of random sign leave z off by 2^-8 sqrt(16 / 3) = 0.009 of its spread: a ReLU then stands on the other side of
    zero in 0.4 x 0.8 x 0.009 of the places, which is sqrt(0.003 / 0.5) = 0.08 of a gradient's norm; four of them."""
    from distributedpytorch_amd.models.xception import XceptionBlock
    torch.manual_seed(0)
    ref = _convert(_weights(XceptionBlock(cin, cout, 3, stride=stride), 1), PLACES[place]).train(training)
    mod = copy.deepcopy(ref).cuda()
    x = torch.randn(2, cin, 19, 23).to(torch.bfloat16)
    xg = x.cuda().contiguous(memory_format=torch.channels_last).requires_grad_(training)
    xr = x.float().requires_grad_(training)
    with torch.set_grad_enabled(training):
        y, want = mod(xg), ref(xr)
    assert y.dtype == torch.bfloat16 and _rel(y, want) < 24 * HALF
    if training:
        dy = torch.randn(want.shape, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
        grads = torch.autograd.grad(y, [xg, *mod.parameters()], dy.cuda().contiguous(memory_format=torch.channels_last))
        wants = torch.autograd.grad(want, [xr, *ref.parameters()], dy.float())
        for name, a, b in zip(["x"] + [n for n, _ in ref.named_parameters()], grads, wants):
            # (what lies before a norm by itself — a depthwise filter of one channel a group, a shift — leaves no gradient)
            if float(b.norm()) > 1e-3 * float(dy.float().norm()):
                assert _rel(a, b) < 48 * HALF + 4 * 0.08, name


def test_xception_converted_after_an_evaluation_keeps_no_folded_constants():
    from distributedpytorch_amd.models.xception import AlignedXception
    torch.manual_seed(0)
    net = AlignedXception(16, 3, pad_mid=False).cuda().eval()
    x = torch.randn(1, 3, 65, 65, device="cuda").to(torch.bfloat16).contiguous(memory_format=torch.channels_last)
    with torch.no_grad():
        net(x)
        ops.convert_group_norm(net)
        first = net(x)[0]
        for m in net.modules():
            if hasattr(m, "eval_refresh"):
                m.eval_refresh()
        assert torch.equal(net(x)[0], first) and torch.isfinite(first).all()
    net.train()
    leaf = x.detach().requires_grad_(True)
    net(leaf)[0].float().square().mean().backward()
    assert all(torch.isfinite(p.grad).all() for p in net.parameters())


@pytest.mark.parametrize("name,classes,channels,layers", [("fcn_resnet18", 21, 3, 22), ("danet_resnet50", 1, 4, 58)])
def test_fcn_and_danet_with_group_norm(name, classes, channels, layers):
    """Evaluation, which computes what training computes without dropout, against fp32 on the CPU: every layer rounds its
    weights, the convolution's map and the norm's, each by at most 2^-8 (spread 2^-8 / sqrt(3)) with random sign; four times the
    spread of their sum.  Then steps of the training engine, eager and captured."""
    from distributedpytorch_amd.models import build_model
    from distributedpytorch_amd.ops import SoftmaxCrossEntropy
    from distributedpytorch_amd.parallel import TrainEngine
    from distributedpytorch_amd.utils import SegmentationMultiLosses
    torch.manual_seed(0)
    ref = build_model(name, classes, in_channels=channels, norm="group").eval()
    x = torch.randn(2, channels, 97, 97, generator=torch.Generator().manual_seed(1))
    with torch.no_grad():
        want = ref(x)
        got = copy.deepcopy(ref).cuda()(x.cuda().to(torch.bfloat16).contiguous(memory_format=torch.channels_last))
    for a, b in zip(*(t if isinstance(t, tuple) else (t,) for t in (got, want))):
        assert _rel(a, b) < 4 * (3 * layers / 3) ** 0.5 * HALF
    y = torch.randint(0, 21, (2, 97, 97), dtype=torch.uint8) if classes > 1 else (torch.rand(2, 1, 97, 97) > 0.5).float()
    for graph_step in (False, True):                       # (no learning: an untrained DANet's logits are in the hundreds)
        crit = SoftmaxCrossEntropy(255) if classes > 1 else SegmentationMultiLosses(1)
        eng = TrainEngine(copy.deepcopy(ref), crit, lr=0.0, momentum=0.0, weight_decay=0.0, device=torch.device("cuda", 0),
                          graph_step=graph_step)
        losses = [float(eng.train_step(x.cuda(), y.cuda())) for _ in range(6)]
        assert all(v == v and v < float("inf") for v in losses) and len(eng._graphs) == int(graph_step), losses
        if not graph_step:
            eng.model.eval()
            crit(eng.ddp(eng.prepare_input(x)), y.cuda()).backward()
            still = [s.name for s in eng.ddp.arena.slots if not s.param.grad.any() or not torch.isfinite(s.param.grad).all()]
            # (DANet's attention branches start with a gain of zero: their projections have no gradient yet)
            assert all(".sa." in n and "_conv" in n for n in still), still
