"""Compiled kernels keep the registers of every lane."""
import os
import re
import shutil
import subprocess
import tempfile

import pytest

from conftest import ROOT
from varlenabsorbflashattn_amd import build as B

CSRC = os.path.join(ROOT, "varlenabsorbflashattn_amd", "csrc")
COPY = re.compile(r"v_accvgpr_write|v_accvgpr_mov|v_mov_b32|v_mov_b64|scratch_store|buffer_store")


def partial_copies(lines):
    """Blocks that copy vector registers and do nothing else before they turn the lanes of a
    branch on again: the lanes that were off there lose what is copied."""
    found, name, block = [], None, None
    for line in lines:
        text = line.split(";")[0].strip()
        if not text:
            continue
        if re.match(r"_Z\w+:", text):
            name, block = text, None
        elif re.match(r"\.LBB\S+:", text):
            block = []
        elif block is None or text.startswith("."):
            continue
        elif re.match(r"s_or_b64 exec, exec,", text):
            copies = [x for x in block if COPY.match(x)]
            others = [x for x in block if not COPY.match(x)
                      and not x.startswith(("s_", "v_writelane", "v_readlane"))]
            if copies and not others:
                found.append((name, copies))
            block = None
        elif "exec" in text or text.startswith(("s_branch", "s_cbranch")):
            block = None
        else:
            block.append(text)
    return found


def test_partial_copies_finds_one():
    bad = ["_Zkernel:", ".LBB0_1:", "\tv_accvgpr_write_b32 a1, v2", "\ts_nop 1",
           "\ts_or_b64 exec, exec, s[0:1]"]
    assert partial_copies(bad) == [("_Zkernel:", ["v_accvgpr_write_b32 a1, v2"])]
    assert not partial_copies(bad[:2] + bad[-1:] + bad[2:-1])
    assert not partial_copies(bad[:3] + ["\tv_add_u32_e32 v0, 1, v0"] + bad[3:])  # a branch's own


@pytest.mark.parametrize("source", [s for s in B.SOURCES if s.endswith(".hip")])
def test_no_copies_of_some_lanes(source):
    try:
        hipcc = B._hipcc()
    except RuntimeError:
        pytest.skip("hipcc not available")
    tmp = tempfile.mkdtemp()
    try:
        out = os.path.join(tmp, "k.s")
        subprocess.run([hipcc, *B._flags(), "--cuda-device-only", "-S", "-o", out,
                        os.path.join(CSRC, source)], check=True, capture_output=True)
        assert not partial_copies(open(out))
    finally:
        shutil.rmtree(tmp, ignore_errors=True)
