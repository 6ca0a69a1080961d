"""GPU: threads with streams of their own share a context (in one process of their own, as test_gpu_transform_tensors.py's checks)."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))


def test_threads_with_streams_of_their_own():
    pytest.importorskip("torch")
    p = subprocess.run([sys.executable, "-u", os.path.join(HERE, "_transform_tensor_threads.py")], capture_output=True, text=True, timeout=100)
    assert "RESULT ok" in p.stdout, p.stdout[-3000:] + p.stderr[-3000:]
