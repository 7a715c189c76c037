"""Models with group norm and with decoder attention on the CPU path: construction, gradients, checkpoints, refusals."""
import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
from distributedpytorch_amd import ops  # noqa: E402
from distributedpytorch_amd.models import build_model  # noqa: E402
from distributedpytorch_amd.models.deeplab import DecoderAttention  # noqa: E402


def test_group_norm_module_is_torchs():
    torch.manual_seed(0)
    gn, ref = ops.GroupNorm2d(12, 4), torch.nn.GroupNorm(4, 12)
    with torch.no_grad():
        for p, q in zip(gn.parameters(), ref.parameters()):
            q.copy_(p.normal_())
    x, r = torch.randn(2, 12, 5, 7), torch.randn(2, 12, 5, 7)
    # fp32 sums of 105 elements in another order
    assert (gn(x, relu=True, residual=r) - torch.relu(ref(x) + r)).abs().max() < 1e-5
    assert set(gn.state_dict()) == set(ref.state_dict())
    gn.eval()
    assert torch.equal(gn(x, dropout=0.5), gn(x))
    gn.train()
    assert (gn(x, dropout=0.5) == 0).float().mean() > 0.3
    with pytest.raises(ValueError):
        ops.GroupNorm2d(48, 32)


def test_convert_group_norm_keeps_parameters_and_divides_the_channels():
    m = build_model("deeplabv3plus_resnet18", 5)
    before = dict(m.named_parameters())
    ops.convert_group_norm(m)
    after = dict(m.named_parameters())
    assert set(before) == set(after) and all(before[k] is after[k] for k in before)
    norms = [t for t in m.modules() if isinstance(t, ops.GroupNorm2d)]
    assert norms and not any(isinstance(t, ops.BatchNorm2d) for t in m.modules())
    assert {(t.num_features, t.num_groups) for t in norms} >= {(48, 16), (64, 32), (256, 32), (512, 32)}


@pytest.mark.parametrize("name,kw", [("deeplabv3plus_resnet18", dict(norm="group", decoder_attention=True)),
                                     ("deeplabv3plus_resnet18", dict(decoder_attention=True)),
                                     ("danet_resnet50", dict(norm="group")), ("fcn_resnet18", dict(norm="group"))])
def test_variants_run_forward_and_backward(name, kw):
    torch.manual_seed(0)
    m = build_model(name, 5, **kw)
    out = m(torch.randn(2, 3, 65, 65))
    outs = out if isinstance(out, tuple) else (out,)
    assert all(t.shape == (2, 5, 65, 65) for t in outs)
    sum(t.float().square().mean() for t in outs).backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in m.parameters())
    one, ten = ({id(p) for p in f()} for f in (m.get_1x_lr_params, m.get_10x_lr_params))
    assert one | ten == {id(p) for p in m.parameters()} and not one & ten
    # one image's result does not depend on the others in evaluation, and with group norm alone not in training either
    m.eval()
    x = torch.randn(2, 3, 65, 65)
    with torch.no_grad():
        both, alone = m(x), m(x[:1])
    both, alone = (t[0] if isinstance(t, tuple) else t for t in (both, alone))
    assert (both[:1] - alone).abs().max() < 1e-3 * alone.abs().max()


def test_decoder_attention_starts_as_the_plain_decoder_and_reaches_every_input():
    torch.manual_seed(1)
    att = DecoderAttention(48, 64, heads=4).eval()
    low, ctx, up = torch.randn(2, 48, 9, 7), torch.randn(2, 64, 5, 3), torch.randn(2, 64, 9, 7)
    assert torch.equal(att(low, ctx, up), up)
    torch.nn.init.ones_(att.norm.weight)
    leaves = [t.requires_grad_(True) for t in (low, ctx, up)]
    y = att(*leaves)
    assert y.shape == up.shape and not torch.equal(y, up)
    grads = torch.autograd.grad(y.square().sum(), leaves + list(att.parameters()))
    assert all(torch.isfinite(g).all() and g.any() for g in grads)


def test_decoder_attention_gradient_against_differences():
    torch.manual_seed(2)
    att = DecoderAttention(4, 32, heads=2).double().eval()
    torch.nn.init.normal_(att.norm.weight)
    args = [torch.randn(1, c, h, w, dtype=torch.float64, requires_grad=True)
            for c, h, w in ((4, 2, 3), (32, 2, 1), (32, 2, 3))]
    assert torch.autograd.gradcheck(att, args)


def test_variant_checkpoint_round_trip_through_the_predictor(tmp_path):
    from distributedpytorch_amd.inference import load_predictor
    import numpy as np
    m = build_model("deeplabv3plus_resnet18", 5, norm="group", decoder_attention=True)
    path = str(tmp_path / "w.pth")
    torch.save(m.state_dict(), path)
    pred = load_predictor("semseg", "deeplabv3plus_resnet18", path, 5, device=torch.device("cpu"), crop=65, batch=1,
                          norm="group", decoder_attention=True)
    out = pred.predict([np.zeros((40, 50, 3), np.uint8)])
    assert out[0].shape == (40, 50)
    with pytest.raises(Exception):
        load_predictor("semseg", "deeplabv3plus_resnet18", path, 5, device=torch.device("cpu"), crop=65, batch=1)


@pytest.mark.parametrize("args,kw,err", [
    (("deeplabv3plus_resnet18", 5), dict(norm="layer"), ValueError),
    (("deeplabv3plus_resnet18", 5), dict(norm="group", sync_bn=True), ValueError),
    (("deeplabv3plus_resnet18", 5), dict(norm="group", freeze_bn=True), ValueError),
    (("deeplabv3plus_xception65", 5), dict(norm="group"), NotImplementedError),
    (("danet_resnet50", 5), dict(decoder_attention=True), ValueError),
])
def test_variant_refusals(args, kw, err):
    with pytest.raises(err):
        build_model(*args, **kw)


def test_convert_group_norm_replaces_the_module_itself_and_shared_ones_once():
    from distributedpytorch_amd import ops
    bn = ops.BatchNorm2d(48)
    gn = ops.convert_group_norm(bn, 32)
    assert isinstance(gn, ops.GroupNorm2d) and gn.num_groups == 16 and gn.weight is bn.weight and gn.bias is bn.bias
    shared = ops.BatchNorm2d(8)
    net = torch.nn.Sequential(shared, torch.nn.Sequential(shared), torch.nn.Identity())
    net.add_module("again", shared)
    out = ops.convert_group_norm(net)
    assert out is net and isinstance(net[0], ops.GroupNorm2d)
    assert net[0] is net[1][0] and net[0] is net.again
    assert len(list(net.parameters())) == 2
