"""The C++ operators (csrc/autograd.cpp) on the CPU: they load against this torch, and refuse what they cannot launch."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from distributedpytorch_amd.csrc import build  # noqa: E402
from distributedpytorch_amd.ops import _backend as B  # noqa: E402


def test_the_library_belongs_to_its_source_and_this_torch():
    assert build.autograd_is_current()
    ops = B.native()
    assert ops is B.native()
    for name in ("group_norm_act", "dropout", "cross_attention"):
        assert getattr(ops, name).default is not None


def test_cpu_tensors_are_refused_before_a_launch():
    ops = B.native()
    x = torch.randn(1, 8, 4, 4).contiguous(memory_format=torch.channels_last)
    q = torch.randn(1, 3, 2, 8, dtype=torch.bfloat16)
    for call in (lambda: ops.group_norm_act.default(x, None, None, None, 2, 1e-5, 0),
                 lambda: ops.dropout.default(x, None, 1000, 1, None, False),
                 lambda: ops.cross_attention.default(q, q, q, None, None, 1.0)):
        with pytest.raises(RuntimeError, match="GPU tensors"):
            call()
    with pytest.raises(RuntimeError, match="an address for each launcher"):
        ops.bind([1, 2])
