"""The three operators as a decoder uses them: group norm, cross attention and dropout in DeepLabv3+ on the GPU."""
import copy
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
pytestmark = pytest.mark.gpu

from distributedpytorch_amd.ops import _backend as B  # noqa: E402


def _rel(got, want):
    return float((got.detach().double().cpu() - want.detach().double()).norm() / want.detach().double().norm())


@pytest.mark.parametrize("low_hw,ctx_hw", [((33, 33), (9, 9)), ((65, 40), (17, 10)), ((8, 8), (1, 1))])
def test_decoder_attention_matches_fp32(low_hw, ctx_hw):
    """Against the same module in fp32 on the CPU.  Every map and weight on the way is rounded once to bf16 (at most 2^-8 of
    its norm): ten of them up to the output, as many again on the way back."""
    from distributedpytorch_amd.models.deeplab import DecoderAttention
    torch.manual_seed(0)
    ref = DecoderAttention(48, 256).eval()
    torch.nn.init.normal_(ref.norm.weight, 1.0, 0.2)
    torch.nn.init.normal_(ref.norm.bias, 0.0, 0.2)
    mod = copy.deepcopy(ref).cuda()
    low, ctx, up = (torch.randn(2, c, *hw).to(torch.bfloat16) for c, hw in ((48, low_hw), (256, ctx_hw), (256, low_hw)))
    dy = torch.randn(2, 256, *low_hw).to(torch.bfloat16)
    cl = torch.channels_last
    gl = [t.cuda().contiguous(memory_format=cl).requires_grad_(True) for t in (low, ctx, up)]
    cpu = [t.float().requires_grad_(True) for t in (low, ctx, up)]
    y, yr = mod(*gl), ref(*cpu)
    assert y.dtype == torch.bfloat16 and y.is_contiguous(memory_format=cl)
    assert _rel(y, yr) < 10 * 2 ** -8
    names = ["low", "context", "up"] + [n for n, _ in ref.named_parameters()]
    got = torch.autograd.grad(y, gl + list(mod.parameters()), dy.cuda().contiguous(memory_format=cl))
    want = torch.autograd.grad(yr, cpu + list(ref.parameters()), dy.float())
    for name, a, b in zip(names, got, want):
        if float(b.norm()) < 1e-3 * float(dy.float().norm()):       # (a key's bias moves every score of a row alike: no gradient)
            continue
        assert _rel(a, b) < 20 * 2 ** -8, name
    n = mod.key_value_conv.out_channels // 2
    kb = got[names.index("key_value_conv.bias")]
    assert float(kb[:n].abs().max()) < 0.05 * float(kb[n:].abs().max())


def _no_dropout(model):
    for m in model.modules():
        if isinstance(getattr(m, "p_drop", None), tuple):
            m.p_drop = (0.0, 0.0)
        elif hasattr(m, "p_drop"):
            m.p_drop = 0.0
    return model


def _model(norm):
    from distributedpytorch_amd.models import build_model
    torch.manual_seed(0)
    m = build_model("deeplabv3plus_resnet50", 21, norm=norm, decoder_attention=True)
    torch.nn.init.ones_(m.decoder.attention.norm.weight)
    return m


@pytest.mark.parametrize("norm", ["batch", "group"])
def test_training_steps_replay_exactly_like_eager_ones(norm):
    from distributedpytorch_amd.ops import SoftmaxCrossEntropy
    from distributedpytorch_amd.parallel import TrainEngine
    base = _no_dropout(_model(norm))
    g = torch.Generator().manual_seed(1)
    xs = [torch.randn(3, 3, 97, 97, generator=g) for _ in range(6)]
    ys = [torch.randint(0, 21, (3, 97, 97), generator=g, dtype=torch.uint8) for _ in range(6)]
    out = {}
    with B.deterministic_mode(True):
        for mode in ("eager", "graph"):
            eng = TrainEngine(copy.deepcopy(base), SoftmaxCrossEntropy(255), lr=0.01, momentum=0.9, weight_decay=1e-4,
                              device=torch.device("cuda", 0), graph_step=mode == "graph")
            losses = [float(eng.train_step(x.cuda(), y.cuda())) for x, y in zip(xs, ys)]
            torch.cuda.synchronize()
            out[mode] = (losses, [p.detach().float().cpu().clone() for p in eng.model.parameters()], len(eng._graphs))
    assert out["eager"][2] == 0 and out["graph"][2] == 1
    assert all(v == v and abs(v) < 1e4 for v in out["eager"][0])
    assert out["eager"][0] == out["graph"][0]
    assert all(torch.equal(a, b) for a, b in zip(out["eager"][1], out["graph"][1]))
    moved = [n for (n, p), q in zip(base.named_parameters(), out["graph"][1]) if not torch.equal(p.detach().float(), q)]
    assert any(n.startswith("decoder.attention.query") for n in moved)


def test_replayed_steps_draw_new_dropout_masks():
    """Only the attention's dropout is on: at learning rate 0 the same batch gives another loss at every replay."""
    from distributedpytorch_amd.ops import SoftmaxCrossEntropy
    from distributedpytorch_amd.parallel import TrainEngine
    m = _no_dropout(_model("group"))
    m.decoder.attention.p_drop = 0.5
    x, y = torch.randn(2, 3, 97, 97).cuda(), torch.randint(0, 21, (2, 97, 97), dtype=torch.uint8).cuda()
    with B.deterministic_mode(True):
        eng = TrainEngine(m, SoftmaxCrossEntropy(255), lr=0.0, momentum=0.0, weight_decay=0.0,
                          device=torch.device("cuda", 0), graph_step=True)
        losses = [float(eng.train_step(x, y)) for _ in range(9)]
    assert len(eng._graphs) == 1 and len(set(losses[4:])) == len(losses[4:]), losses


@pytest.mark.parametrize("norm", ["batch", "group"])
def test_prediction_replays_like_the_eager_forward(norm):
    from distributedpytorch_amd.parallel.graphs import GraphedForward
    m = _model(norm).cuda().eval()
    graphed = GraphedForward(m)
    with torch.no_grad():
        for seed in range(3):
            x = torch.randn(1, 3, 97, 97, generator=torch.Generator().manual_seed(seed)).cuda().to(torch.bfloat16)
            x = x.contiguous(memory_format=torch.channels_last)
            want = m(x)
            assert torch.equal(graphed(x), want), seed
