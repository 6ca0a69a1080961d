"""Runs in a process of its own, where torch is imported before lnasr's library: how much memory a context keeps behind a call.
Prints RESULT ok, or what went wrong."""
import os
import sys

import numpy as np
import torch

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path[:0] = [HERE, os.path.join(os.path.dirname(HERE), "ln-asr_amd")]
from lnasr import _ffi, transform  # noqa: E402


def main():
    """256 groups of 1024 x 1024 sums, one of them long: 32-bit sums are kept for its spans only."""
    c = _ffi.Context(0)
    G, I, O, long = 256, 1024, 1024, 4000
    sizes = np.full(G, 2)
    sizes[77] = long
    off = torch.from_numpy(np.concatenate([[0], np.cumsum(sizes)])).cuda()
    F = int(sizes.sum())
    x, dy = torch.randn(F, I, device="cuda"), torch.randn(F, O, device="cuda")
    w, out = torch.zeros(G, O, I, device="cuda"), {"w": torch.zeros(G, O, I, device="cuda"), "bias": torch.zeros(G, O, device="cuda")}
    transform.affine_grad(x[:3, :5], torch.tensor([0, 3], device="cuda"), w[:1, :4, :5].contiguous(), dy[:3, :4], out={"w": torch.zeros(1, 4, 5, device="cuda")}, ctx=c)
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    transform.affine_grad(x, off, w, dy, out=out, ctx=c)
    torch.cuda.synchronize()
    kept = before - torch.cuda.mem_get_info()[0]
    assert kept < 256 << 20, "%d MB kept" % (kept >> 20)
    for g in (0, 76, 77, 78, 255):
        lo, hi = int(off[g]), int(off[g + 1])
        want = dy[lo:hi].double().T @ x[lo:hi].double()
        bound = (hi - lo + 4) * 2.0 ** -24 * (dy[lo:hi].double().abs().T @ x[lo:hi].double().abs()) + 2.0 ** -24 * want.abs()
        assert bool(((out["w"][g].double() - want).abs() <= bound).all()), g
    print("RESULT ok", flush=True)


if __name__ == "__main__":
    main()
