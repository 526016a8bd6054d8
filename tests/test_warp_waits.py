"""Waits on barriers in the group-scaled products' kernels, read from their
source.  A wait gives up after a number of tries, and lanes of a warp may come
to different answers; so a wait whose answer a whole warp acts on (warp-wide
instructions follow) has to be the voting form, mbar_wait_warp, and the plain
form stays with code that one lane runs alone."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mojostream_b200", "csrc")


def code(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def waits(text):
    """(line, heads of the blocks around it) of every plain mbar_wait."""
    heads, start, found = [], 0, []
    for m in re.finditer(r"[{};]|\bmbar_wait\(", text):
        t = m.group()
        if t == "{":
            heads.append(text[start:m.start()].strip())
        elif t == "}":
            heads.pop()
        elif t != ";":
            found.append((text.count("\n", 0, m.start()) + 1, list(heads)))
            continue
        start = m.end()
    assert not heads
    return found


@pytest.mark.parametrize("name", ["ms_q4g.cu", "ms_q4g_tc.cu"])
def test_plain_waits_are_one_lanes_own(name):
    text = code(name)
    assert "mbar_wait_warp(" in text
    for line, heads in waits(text):
        assert any(re.search(r"if \(lane == 0\)$", h) for h in heads), f"{name}:{line}"


def test_the_voting_form_votes():
    body = code("ms_common.cuh").split("mbar_wait_warp(", 1)[1].split("}", 1)[0]
    assert re.search(r"__all_sync\(0xffffffffu, mbar_wait\(bar, parity\)\)", body)
