"""GPU: feature transforms inside a torch.autograd.Function, and refused outside of one (in a process of their own, as
test_gpu_transform_tensors.py's checks)."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))


def test_the_halves_of_a_function():
    pytest.importorskip("torch")
    p = subprocess.run([sys.executable, "-u", os.path.join(HERE, "_transform_autograd.py")], capture_output=True, text=True, timeout=100)
    assert "RESULT ok" in p.stdout, p.stdout[-3000:] + p.stderr[-3000:]
