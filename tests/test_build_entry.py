"""The build entry point: everything by default and under DPAMD_BUILD_FORCE=1, what has changed with force=False."""
import os
import sys

import pytest

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import __graft_entry__  # noqa: E402
from distributedpytorch_amd.csrc import build  # noqa: E402


@pytest.mark.parametrize("kw,env,want", [({}, None, True), ({}, "0", True), ({"force": False}, None, False),
                                         ({"force": False}, "0", False), ({"force": False}, "1", True)])
def test_what_build_compiles(kw, env, want, monkeypatch):
    asked = []
    monkeypatch.setattr(build, "build_all", lambda force=False, verbose=False: asked.append(force) or force)
    monkeypatch.delenv("DPAMD_BUILD_FORCE", raising=False)
    if env is not None:
        monkeypatch.setenv("DPAMD_BUILD_FORCE", env)
    __graft_entry__.build(**kw)
    assert asked == [want]
