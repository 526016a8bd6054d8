"""Whose the operators' workspaces are (mojostream_b200/csrc/ms_ws.h), checked on
the host: tests/ws_pool_check.cc drives the pool through random calls on streams
and into graphs against a pretended device."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_no_two_hold_one_workspace(tmp_path):
    exe = tmp_path / "ws_pool_check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror",
                    "-I", os.path.join(ROOT, "mojostream_b200", "csrc"),
                    os.path.join(ROOT, "tests", "ws_pool_check.cc"), "-o", str(exe)],
                   check=True, capture_output=True, text=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stdout[-2000:] + out.stderr[-2000:]
    assert out.stdout.strip().endswith("ok")
