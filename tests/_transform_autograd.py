"""Runs in a process of its own, where torch is imported before lnasr's library: the feature transforms as the two halves of a
torch.autograd.Function.  Prints RESULT ok, or what went wrong."""
import os
import sys

import numpy as np
import torch

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path[:0] = [HERE, os.path.join(os.path.dirname(HERE), "ln-asr_amd")]
import _transform_ref as ref  # noqa: E402
from lnasr import _ffi, transform  # noqa: E402


class Projection(torch.autograd.Function):
    @staticmethod
    def forward(c, x, w, a, b, bias, offsets, scale, slots):
        c.save_for_backward(x, w, a, b, offsets, scale, slots)
        return transform.projection(x, offsets, w, a, b, bias, scale, slots)

    @staticmethod
    def backward(c, dy):
        x, w, a, b, offsets, scale, slots = c.saved_tensors
        g = transform.projection_grad(x, offsets, w, a, b, dy.contiguous(), scale, slots)
        return g["x"], g["w"], g["a"], g["b"], g["bias"], None, None, None


def main():
    d = ref.make(50, (700, 72, 80, 6, 4, 16), negative=True)
    names = ("x", "w", "a", "b", "bias")
    t = {k: torch.from_numpy(d[k]).cuda().requires_grad_() for k in names}
    rest = [torch.from_numpy(d[k]).cuda() for k in ("offsets", "scale", "slots")]
    try:
        transform.projection(t["x"], rest[0], t["w"], t["a"], t["b"], t["bias"], rest[1], rest[2])
    except _ffi.LnasrError as e:
        assert "x requires a gradient" in str(e), e
    else:
        raise AssertionError("taken, and its graph lost")
    y = Projection.apply(*(t[k] for k in names), *rest)
    want, err = ref.projection("float64", d["x"], d["offsets"], d["w"], d["a"], d["b"], d["bias"], d["scale"], d["slots"], d["y0"])
    ref.check(y.detach().cpu().numpy(), want, err, "y")
    y.backward(torch.from_numpy(d["dy"]).cuda())                          # (backward runs in a thread of torch's)
    want, err = ref.projection_grad("float64", d["x"], d["offsets"], d["w"], d["a"], d["b"], d["dy"], d["scale"], d["slots"], d["dx0"])
    for k in names:
        ref.check(t[k].grad.cpu().numpy(), want[k], err[k], k)
    with torch.no_grad():
        z = transform.projection(t["x"], rest[0], t["w"], t["a"], t["b"], t["bias"], rest[1], rest[2])
    assert torch.equal(z, y)
    print("RESULT ok", flush=True)


if __name__ == "__main__":
    main()
