"""Runs in a process of its own, where torch is imported before lnasr's library: threads that share a context, each with a stream of
its own or with none.  Prints RESULT ok, or what went wrong."""
import os
import sys
import threading
import traceback

import torch

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path[:0] = [HERE, os.path.join(os.path.dirname(HERE), "ln-asr_amd")]
import _transform_ref as ref  # noqa: E402
from lnasr import _ffi, transform  # noqa: E402


def main():
    ctx = _ffi.Context(0)
    size = (3000, 72, 80, 5, 5, 8)
    data = []
    for i in range(3):
        d = ref.make(40 + i, size, slots=False)
        t = {k: torch.from_numpy(d[k]).cuda().to(torch.float32) for k in ("x", "w3", "bias2")}
        t["offsets"] = torch.from_numpy(d["offsets"]).cuda()
        h = {k: t[k].double().cpu().numpy() for k in ("x", "w3", "bias2")}
        data.append((t, ref.affine("float32", h["x"], d["offsets"], h["w3"], h["bias2"], None, d["y0"])))
    torch.cuda.synchronize()
    failed, gate = [], threading.Barrier(3)

    def work(i):
        try:
            t, (want, bound) = data[i]
            s = torch.cuda.Stream()
            slow = torch.randn(2048, 2048, device="cuda")
            late = torch.zeros_like(t["x"])
            torch.cuda.synchronize()
            for turn in range(10):
                gate.wait(60)
                with torch.cuda.stream(s):
                    if i < 2:                                              # (the third thread chooses none)
                        ctx.use_stream(s)
                    gate.wait(60)                                          # every thread has chosen before any calls
                    late.zero_()
                    for _ in range(10):
                        slow = slow @ slow * 1e-3
                    late.copy_(t["x"])
                    y = transform.affine(late, t["offsets"], t["w3"], t["bias2"], ctx=ctx)
                    z = y + 0
                s.synchronize()
                ref.check(z.double().cpu().numpy(), want, bound, "thread %d turn %d" % (i, turn))
        except Exception:
            failed.append(traceback.format_exc())
            gate.abort()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    print("RESULT", "ok" if not failed else "\n".join(failed), flush=True)


if __name__ == "__main__":
    main()
