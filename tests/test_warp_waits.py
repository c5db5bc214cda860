"""CPU: a warp that learns from one of its lanes that an mbarrier has completed needs a barrier of its own before the
other lanes read what was loaded: every such wait of the kernels goes through mbar_wait_warp (csrc/s2_common.cuh), which
has it."""
import os
import re

from tests.conftest import ROOT

CSRC = os.path.join(ROOT, "seedvr2_ncnn_b200", "csrc")


def _sources():
    return {f: open(os.path.join(CSRC, f)).read() for f in sorted(os.listdir(CSRC)) if f.endswith((".cu", ".cuh"))}


def test_one_lane_waits_only_in_mbar_wait_warp():
    found = 0
    for f, text in _sources().items():
        for m in re.finditer(r"= mbar_wait(<\w+>)?\([^;]*\? 1 : 0;", text):  # one lane's answer for the others
            assert f == "s2_common.cuh", f"{f}:{text.count(chr(10), 0, m.start()) + 1}"
            found += 1
    assert found == 1


def test_mbar_wait_warp_orders_memory():
    text = _sources()["s2_common.cuh"]
    body = text[text.index("bool mbar_wait_warp("):]
    body = body[:body.index("\n}")]
    assert body.index("__shfl_sync") < body.index("__syncwarp();") < body.index("return")
