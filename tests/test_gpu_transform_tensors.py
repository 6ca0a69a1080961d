"""GPU: feature transforms on tensors of another library (torch's), in one process of their own: torch has to be imported before lnasr's
library there, and the other tests of this suite run without it.  The checks are _transform_tensors.py's."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))
CHECKS = ["bfloat16", "bfloat16_wide", "strides", "streams", "graphs", "far_rows", "unchosen_streams", "pinned", "graph_outlives_context"]


@pytest.fixture(scope="module")
def results():
    pytest.importorskip("torch")
    p = subprocess.run([sys.executable, "-u", os.path.join(HERE, "_transform_tensors.py")] + CHECKS, capture_output=True, text=True, timeout=100)
    said = {}
    for line in p.stdout.splitlines():
        if line.startswith("RESULT "):
            said[line.split()[1]] = line.split()[2]
    return said, p.stdout[-3000:] + p.stderr[-3000:]


@pytest.mark.parametrize("check", CHECKS)
def test_tensors(results, check):
    said, tail = results
    assert said.get(check) == "ok", tail
