"""GPU: workspaces of the feature transforms (in a process of their own, as test_gpu_transform_tensors.py's checks)."""
import os
import subprocess
import sys

import numpy as np
import pytest

import _transform_ref as ref

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))


def test_sums_are_kept_for_long_groups_only():
    pytest.importorskip("torch")
    p = subprocess.run([sys.executable, "-u", os.path.join(HERE, "_transform_memory.py")], capture_output=True, text=True, timeout=100)
    assert "RESULT ok" in p.stdout, p.stdout[-3000:] + p.stderr[-3000:]


@pytest.mark.parametrize("kind", ["float64", "float32", "float16"])
@pytest.mark.parametrize("I,O", [(39, 39), (130, 72)])
def test_groups_of_every_number_of_spans(kind, I, O):
    """More groups than spans and fewer: groups that begin anywhere in a span, of one span, of several, of none."""
    from lnasr import _ffi
    ctx = _ffi.Context(0)
    rng = np.random.default_rng(5)
    for G, most in ((300, 40), (5, 9000)):
        sizes = rng.integers(0, most, G)
        sizes[G // 2] = 20011
        sizes[G // 2 + 1] = 0
        sizes[G // 2 + 2] = 5000
        off = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int64)
        F = int(off[-1])
        x, dy = rng.standard_normal((F, I)).astype(kind), rng.standard_normal((F, O)).astype(kind)
        w = np.zeros((G, O, I), kind)
        for slots in (None, rng.permutation(G).astype(np.int32)):
            got = ctx.affine_grad(x, off, w, dy, slots, want=("w", "bias"))
            want, err = ref.affine_grad(kind, x, off, w, dy, slots, np.zeros((F, I)))
            for k in got:
                ref.check(got[k], want[k], err[k], k)
    ctx.close()
