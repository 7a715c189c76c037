"""The assembly of the attention kernels: no path reads a matrix instruction's result before it is written.

gfx950 does not interlock ordinary vector instructions with the results of v_mfma: the compiler keeps the distance, by
instructions between or by s_nop.  Where a branch joined again between the two it was found to count the longer way only,
and the shorter one read registers too early — now and then, and only in some launches.  The kernels are written so that
no branch stands there; this test reads what the compiler made of them and counts the shortest way."""
import os
import re
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
from distributedpytorch_amd.csrc import build  # noqa: E402


def _registers(text):
    out = set()
    for m in re.finditer(r"\b([va])\[(\d+):(\d+)\]|\b([va])(\d+)\b", text):
        out |= {m[1] + str(i) for i in range(int(m[2]), int(m[3]) + 1)} if m[1] else {m[4] + m[5]}
    return out


def _waits(op):
    """Wait states between a matrix instruction and an ordinary one that touches its result: passes + 3 (32x32x16: 8
    passes, 16x16x32: 4 passes; the slower ones of one 32-row tile: 16)."""
    if "32x32x16" in op:
        return 11
    return 7 if "16x16x32" in op else 19


def _kernels(lines):
    name, body, out = None, None, {}
    for line in lines:
        line = line.split(";")[0].rstrip()
        if m := re.match(r"^(\w+):", line):
            if not line.startswith(".L"):
                name, body = m[1], []
                out[name] = body
        if body is None:
            continue
        if m := re.match(r"^(\.LBB\w+):", line):
            body.append((m[1], None, None))
        elif m := re.match(r"^\s+([a-z]\w+)\s*(.*)$", line):
            body.append((None, m[1], m[2]))
            if m[1] == "s_endpgm":
                body = None
    return out


def early_touches(lines):
    """[(kernel, matrix instruction, instruction that reads or writes its result too early, wait states between)]"""
    found = []
    for name, body in _kernels(lines).items():
        labels = {label: i for i, (label, _, _) in enumerate(body) if label}
        for start, (_, op, args) in enumerate(body):
            if not op or not op.startswith("v_mfma"):
                continue
            dst, need = _registers(args.split(",")[0]), _waits(op)
            seen, todo = {}, [(start + 1, 0)]
            while todo:
                i, w = todo.pop()
                if w >= need or i >= len(body) or seen.get(i, need) <= w:
                    continue
                seen[i] = w
                label, op2, args2 = body[i]
                if label:
                    todo.append((i + 1, w))
                elif op2.startswith("s_branch"):
                    todo.append((labels[args2.strip()], w + 1))
                elif op2.startswith("s_cbranch"):
                    todo += [(labels[args2.strip()], w + 1), (i + 1, w + 1)]
                elif op2.startswith("v_mfma"):
                    d, a, b, c = (_registers(t) for t in re.split(r",\s*", args2)[:4])
                    if (a | b) & dst:
                        found.append((name, args, op2 + " " + args2, w))
                    elif d != dst and c != dst:          # (an accumulation in place waits by itself)
                        todo.append((i + 1, w + 1))
                elif op2.startswith(("v_", "ds_write", "global_store", "buffer_store", "scratch_store", "global_atomic")) and \
                        _registers(args2) & dst:
                    found.append((name, args, op2 + " " + args2, w))
                elif op2 != "s_endpgm":
                    todo.append((i + 1, w + (int(args2.split()[0], 0) + 1 if op2 == "s_nop" else 1)))
    return found


MFMA = "\tv_mfma_f32_32x32x16_bf16 v[0:15], v[16:19], v[20:23], 0"


@pytest.mark.parametrize("between,early", [
    (["\ts_nop 9"], True), (["\ts_nop 10"], False), (["\tv_mov_b32_e32 v40, v41"] * 11, False),
    # the short way round a block that is long enough by itself
    (["\ts_cbranch_scc1 .LBB0_1"] + ["\tv_mov_b32_e32 v40, v41"] * 12 + [".LBB0_1:"], True),
    (["\ts_cbranch_scc1 .LBB0_1"] + ["\tv_mov_b32_e32 v40, v41"] * 12 + [".LBB0_1:", "\ts_nop 9"], False)])
def test_the_reader_counts_the_shortest_way(between, early):
    lines = ["kernel:", MFMA, *between, "\tv_mul_f32_e32 v50, v3, v51", "\ts_endpgm"]
    assert bool(early_touches(lines)) == early


@pytest.mark.skipif(not os.path.isfile(build.HIPCC), reason="needs hipcc")
@pytest.mark.parametrize("source", ["cross_attention.hip", "attention.hip"])
def test_no_early_touch(source, tmp_path):
    out = tmp_path / "kernels.s"
    flags = [f for f in build.hip_flags(source) if f not in ("-shared", "-c")]
    path = os.path.join(ROOT, "distributedpytorch_amd", "csrc", source)
    subprocess.run([build.HIPCC, *flags, "-S", "--cuda-device-only", path, "-o", str(out)], check=True, capture_output=True)
    lines = out.read_text().splitlines()
    assert sum(line.lstrip().startswith("v_mfma") for line in lines) > 100
    assert early_touches(lines) == []
