"""Contexts that several threads make at the same time."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_contexts_of_several_threads_plan_alike():
    """What the launch plans ask of the driver once is complete before any
    context uses it: every thread's product has the same bits, those that a
    process with one thread gets."""
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    bits = set()
    for n in (1, 6, 6):
        out = subprocess.run([sys.executable, os.path.join(ROOT, "tests", "context_worker.py"), str(n)],
                             capture_output=True, text=True, timeout=300, cwd=ROOT,
                             env=dict(os.environ, PYTHONPATH=ROOT))
        assert out.returncode == 0, out.stderr[-2000:]
        assert len(out.stdout.split()) == n
        bits |= set(out.stdout.split())
    assert len(bits) == 1
