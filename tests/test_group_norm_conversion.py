"""convert_group_norm on Xception: stored at its own width it is converted, stored wider it is refused (CPU)."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from distributedpytorch_amd import ops  # noqa: E402
from distributedpytorch_amd.models import xception  # noqa: E402


@pytest.mark.parametrize("part", ["whole", "middle", "a block", "a layer"])
def test_a_flow_that_is_stored_wider_is_refused_and_left_alone(part):
    net = xception.AlignedXception(16, 3, pad_mid=True)
    module = {"whole": net, "middle": net.middle, "a block": net.block20, "a layer": net.block3.skipbn}[part]
    before = {n: type(m) for n, m in net.named_modules()}
    with pytest.raises(NotImplementedError, match="wider"):
        ops.convert_group_norm(module)
    assert {n: type(m) for n, m in net.named_modules()} == before


def test_a_flow_of_its_own_width_is_converted():
    net = ops.convert_group_norm(xception.AlignedXception(16, 3, pad_mid=False))
    assert not any(isinstance(m, ops.BatchNorm2d) for m in net.modules())
    assert {m.num_groups for m in net.modules() if isinstance(m, ops.GroupNorm2d) and m.num_features == 728} == {8}
    # parts of the padded model that hold no padding are converted too
    padded = xception.AlignedXception(16, 3, pad_mid=True)
    assert ops.convert_group_norm(padded.block2) is padded.block2
    assert isinstance(padded.block2.skipbn, ops.GroupNorm2d)
    x = torch.randn(1, 3, 33, 33)
    out, low = net(x)
    (out.square().mean() + low.square().mean()).backward()
    assert all(torch.isfinite(p.grad).all() for p in net.parameters())
