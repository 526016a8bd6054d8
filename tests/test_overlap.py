"""Which operands share memory (mojostream_b200/csrc/ms_overlap.h), checked on
the host: tests/overlap_check.cc compares it with a map of bytes."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_rows_that_share_memory(tmp_path):
    exe = tmp_path / "overlap_check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror",
                    "-I", os.path.join(ROOT, "mojostream_b200", "csrc"),
                    os.path.join(ROOT, "tests", "overlap_check.cc"), "-o", str(exe)],
                   check=True, capture_output=True, text=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stdout[-2000:] + out.stderr[-2000:]
    assert out.stdout.strip().endswith("ok")
