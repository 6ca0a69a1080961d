"""Runs in a process of its own (test_gpu_transform_tensors.py), where torch is imported before lnasr's library, so that both use one
HIP runtime: the feature transforms on tensors -- bfloat16, strides and alignments, streams, graphs, far offsets.  Prints one line for
each check that was asked for: its name and "ok", or what went wrong."""
import os
import sys
import traceback

import numpy as np
import torch

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path[:0] = [HERE, os.path.join(os.path.dirname(HERE), "ln-asr_amd")]
import _transform_ref as ref  # noqa: E402
from lnasr import _ffi, transform  # noqa: E402

ctx = transform.default_ctx()
TYPES = {"float64": torch.float64, "float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def up(d, kind):
    """The inputs as tensors of the type, and as the float64 values those hold."""
    t = {k: None if v is None else torch.from_numpy(v).cuda() if k in ("offsets", "slots", "scale") else torch.from_numpy(v).cuda().to(TYPES[kind])
         for k, v in d.items()}
    h = {k: d[k] if k in ("offsets", "slots", "scale") else v.double().cpu().numpy() for k, v in t.items()}
    torch.cuda.synchronize()
    return t, h


def host(t):
    return t.double().cpu().numpy()


def both(kind, size, seed, shared=True, **kw):
    """Both operators and their gradients at one size."""
    t, h = up(ref.make(seed, size, **kw), kind)
    y = transform.affine(t["x"], t["offsets"], t["w3"], t["bias2"], t["slots"], out=t["y0"].clone())
    torch.cuda.synchronize()
    ref.check(host(y), *ref.affine(kind, h["x"], h["offsets"], h["w3"], h["bias2"], h["slots"], h["y0"]), "affine")
    g = transform.affine_grad(t["x"], t["offsets"], t["w3"], t["dy"], t["slots"])
    torch.cuda.synchronize()
    want, err = ref.affine_grad(kind, h["x"], h["offsets"], h["w3"], h["dy"], h["slots"], h["dx0"])
    for k in want:
        ref.check(host(g[k]), want[k], err[k], "affine_grad " + k)
    if kw.get("slots", True):
        t["slots"][::3] = -1
        h["slots"] = t["slots"].cpu().numpy()
    y = transform.projection(t["x"], t["offsets"], t["w"], t["a"], t["b"], t["bias"], t["scale"], t["slots"])
    torch.cuda.synchronize()
    ref.check(host(y), *ref.projection(kind, h["x"], h["offsets"], h["w"], h["a"], h["b"], h["bias"], h["scale"], h["slots"], h["y0"]), "projection")
    names = ("x", "a", "b", "w", "bias") if shared else ("x", "a", "b")
    g = transform.projection_grad(t["x"], t["offsets"], t["w"], t["a"], t["b"], t["dy"], t["scale"], t["slots"], want=names)
    torch.cuda.synchronize()
    want, err = ref.projection_grad(kind, h["x"], h["offsets"], h["w"], h["a"], h["b"], h["dy"], h["scale"], h["slots"], h["dx0"])
    assert tuple(g) == names
    for k in names:
        ref.check(host(g[k]), want[k], err[k], "projection_grad " + k)


def bfloat16():
    for i, size in enumerate(ref.SIZES):
        print("  ", size, flush=True)
        both("bfloat16", size, i)
        both("bfloat16", size, i + 100, slots=False)
        both("bfloat16", size, i + 200, single=True)


def bfloat16_wide():
    """The 256 x 256 tiles in both directions and for sums: long and short k, uneven edges, a segment's end inside a tile."""
    for i, (size, kw) in enumerate((((9001, 840, 2056, 5, 4, 24), {}), ((17000, 72, 1032, 3, 2, 40), {}), ((16500, 1030, 270, 9, 3, 9), {}),
                                    ((24000, 512, 520, 40, 32, 16), {"empties": False}), ((24000, 513, 600, 33, 32, 8), {"slots": False}))):
        print("  ", size, flush=True)
        both("bfloat16", size, 300 + i, **kw)


def strides():
    """x and y are columns of wider tensors whose other columns hold NaN, or start off any alignment; the columns around y stay."""
    for kind in TYPES:
        for F, I, O in ((70, 39, 24), (300, 64, 130), (5, 256, 40)):
            d = ref.make(1, (F, I, O, 4, 3, 8))
            t, h = up(d, kind)
            for left, right in ((0, 5), (8, 8), (3, 2), (1, 0)):
                x = torch.full((F, left + I + right), float("nan"), device="cuda", dtype=TYPES[kind])
                x[:, left:left + I] = t["x"]
                y = torch.full((F, left + O + right), 7.0, device="cuda", dtype=TYPES[kind])
                dy = torch.full((F, left + O + right), float("nan"), device="cuda", dtype=TYPES[kind])
                dy[:, left:left + O] = t["dy"]
                dx = torch.full((F, left + I + right), 7.0, device="cuda", dtype=TYPES[kind])
                torch.cuda.synchronize()
                xs, ys, dys, dxs = x[:, left:left + I], y[:, left:left + O], dy[:, left:left + O], dx[:, left:left + I]
                transform.affine(xs, t["offsets"], t["w3"], t["bias2"], t["slots"], out=ys)
                g = transform.affine_grad(xs, t["offsets"], t["w3"], dys, t["slots"],
                                          out={"x": dxs, "w": torch.empty_like(t["w3"]), "bias": torch.empty_like(t["bias2"])})
                torch.cuda.synchronize()
                ref.check(host(ys), *ref.affine(kind, h["x"], h["offsets"], h["w3"], h["bias2"], h["slots"], h["y0"]), "y")
                want, err = ref.affine_grad(kind, h["x"], h["offsets"], h["w3"], h["dy"], h["slots"], h["dx0"])
                for k in want:
                    ref.check(host(g[k]), want[k], err[k], k)
                y[:, left:left + O] = 7.0
                dx[:, left:left + I] = 7.0
                assert bool((y == 7.0).all()) and bool((dx == 7.0).all())
                y0 = torch.full_like(y, 7.0)
                torch.cuda.synchronize()
                transform.projection(xs, t["offsets"], t["w"], t["a"], t["b"], t["bias"], t["scale"], t["slots"], out=y0[:, left:left + O])
                g = transform.projection_grad(xs, t["offsets"], t["w"], t["a"], t["b"], dys, t["scale"], t["slots"])
                torch.cuda.synchronize()
                ref.check(host(y0[:, left:left + O]),
                          *ref.projection(kind, h["x"], h["offsets"], h["w"], h["a"], h["b"], h["bias"], h["scale"], h["slots"], h["y0"]), "projection")
                want, err = ref.projection_grad(kind, h["x"], h["offsets"], h["w"], h["a"], h["b"], h["dy"], h["scale"], h["slots"], h["dx0"])
                for k in want:
                    ref.check(host(g[k]), want[k], err[k], k)
                y0[:, left:left + O] = 7.0
                assert bool((y0 == 7.0).all())
    # matrices that begin anywhere
    t, h = up(ref.make(2, (200, 72, 136, 3, 3, 16), slots=False), "bfloat16")
    for k in ("w3", "w", "a", "b"):
        room = torch.empty(t[k].numel() + 1, device="cuda", dtype=torch.bfloat16)
        room[1:] = t[k].flatten()
        t[k] = room[1:].view(t[k].shape)
    torch.cuda.synchronize()
    y = transform.affine(t["x"], t["offsets"], t["w3"], t["bias2"])
    z = transform.projection(t["x"], t["offsets"], t["w"], t["a"], t["b"])
    torch.cuda.synchronize()
    ref.check(host(y), *ref.affine("bfloat16", h["x"], h["offsets"], h["w3"], h["bias2"], None, h["y0"]))
    ref.check(host(z), *ref.projection("bfloat16", h["x"], h["offsets"], h["w"], h["a"], h["b"], None, None, None, h["y0"]))
    for bad, what in ((t["x"].t().contiguous().t(), "x"), (t["w3"].transpose(1, 2).contiguous().transpose(1, 2), "w")):
        try:
            transform.affine(bad if what == "x" else t["x"], t["offsets"], bad if what == "w" else t["w3"])
        except _ffi.LnasrError as e:
            assert "contiguous" in str(e) and e.args[0].startswith(what), e
        else:
            raise AssertionError("columns for rows were taken")


def streams():
    """Inputs made on another stream just before the call: in order where the context works on that stream."""
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    t, h = up(ref.make(3, (4000, 64, 48, 5, 5, 8), slots=False), "float32")
    want, bound = ref.affine("float32", h["x"], h["offsets"], h["w3"], h["bias2"], None, h["y0"])
    late, slow = torch.zeros_like(t["x"]), torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    for s in (s1, s2, s1, torch.cuda.default_stream()):
        ctx.use_stream(s)
        with torch.cuda.stream(s):
            late.zero_()
            for _ in range(20):
                slow = slow @ slow * 1e-3
            late.copy_(t["x"])
            y = transform.affine(late, t["offsets"], t["w3"], t["bias2"])
            z = y + 0                                                   # read on the same stream, without a wait
        torch.cuda.synchronize()
        ref.check(host(z), want, bound)
    ctx.use_stream(None)
    y = transform.affine(late, t["offsets"], t["w3"], t["bias2"])
    ctx.sync()
    ref.check(host(y), want, bound)
    assert torch.cuda.current_device() == 0
    # two contexts at once, each on a stream of its own, with workspaces of their own
    other = _ffi.Context(0)
    ctx.use_stream(s1)
    other.use_stream(s2)
    t2, h2 = up(ref.make(4, (3000, 72, 40, 4, 3, 16)), "bfloat16")
    t3, h3 = up(ref.make(5, (3000, 72, 40, 4, 3, 16)), "bfloat16")
    for _ in range(5):
        a = transform.projection_grad(t2["x"], t2["offsets"], t2["w"], t2["a"], t2["b"], t2["dy"], t2["scale"], t2["slots"], ctx=ctx)
        b = transform.projection_grad(t3["x"], t3["offsets"], t3["w"], t3["a"], t3["b"], t3["dy"], t3["scale"], t3["slots"], ctx=other)
        torch.cuda.synchronize()
        for got, q in ((a, h2), (b, h3)):
            w, e = ref.projection_grad("bfloat16", q["x"], q["offsets"], q["w"], q["a"], q["b"], q["dy"], q["scale"], q["slots"], q["dx0"])
            for k in w:
                ref.check(host(got[k]), w[k], e[k], k)
    ctx.use_stream(None)
    other.close()


def graphs():
    """A captured run of all four calls, replayed on new inputs with eager calls between, gives what eager calls give, bit by bit --
    after the context's workspaces had to grow, too."""
    c = _ffi.Context(0)
    s = torch.cuda.Stream()
    c.use_stream(s)
    size = (3000, 80, 136, 6, 4, 16)
    t, _ = up(ref.make(6, size), "bfloat16")
    out = {"y": torch.zeros_like(t["y0"]), "p": torch.zeros_like(t["y0"])}
    ga = {"x": torch.zeros_like(t["x"]), "w": torch.zeros_like(t["w3"]), "bias": torch.zeros_like(t["bias2"])}
    gp = {k: torch.zeros_like(t[k]) for k in ("x", "a", "b", "w", "bias")}

    def everything(y, p, a, b):
        transform.affine(t["x"], t["offsets"], t["w3"], t["bias2"], t["slots"], out=y, ctx=c)
        transform.affine_grad(t["x"], t["offsets"], t["w3"], t["dy"], t["slots"], out=a, ctx=c)
        transform.projection(t["x"], t["offsets"], t["w"], t["a"], t["b"], t["bias"], t["scale"], t["slots"], out=p, ctx=c)
        transform.projection_grad(t["x"], t["offsets"], t["w"], t["a"], t["b"], t["dy"], t["scale"], t["slots"], out=b, ctx=c)

    with torch.cuda.stream(s):
        fresh = torch.cuda.CUDAGraph()
        refused = None
        with torch.cuda.graph(fresh, stream=s):
            try:
                transform.projection(t["x"], t["offsets"], t["w"], t["a"], t["b"], slots=t["slots"], out=out["p"], ctx=c)
            except _ffi.LnasrError as e:
                refused = str(e)
            (out["y"] + 1).sum()                                          # (an empty capture is an error of its own)
        assert refused and "run the call once before" in refused, refused
        everything(out["y"], out["p"], ga, gp)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        said = []
        with torch.cuda.graph(graph, stream=s):
            everything(out["y"], out["p"], ga, gp)
            for call in (lambda: c.use_stream(None), lambda: transform.affine(t["x"], np.array([0, 3000]), t["w3"][:1], out=out["y"], ctx=c)):
                try:
                    call()
                except _ffi.LnasrError as e:
                    said.append(str(e))
        assert "being captured" in said[0] and "host array" in said[1], said
        eager = (torch.zeros_like(out["y"]), torch.zeros_like(out["p"]), {k: torch.zeros_like(v) for k, v in ga.items()},
                 {k: torch.zeros_like(v) for k, v in gp.items()})
        for turn in range(4):
            new, _ = up(ref.make(20 + turn, size), "bfloat16")
            for k in ("x", "dy", "w3", "w", "a", "b", "slots", "offsets"):
                t[k].copy_(new[k])
            for v in (out["y"], out["p"], *ga.values(), *gp.values()):
                v.fill_(3.0)
            graph.replay()
            torch.cuda.synchronize()
            if turn == 1:                                                  # a larger call: the workspaces grow
                big, hb = up(ref.make(9, (20000, 80, 136, 6, 4, 64)), "bfloat16")
                y = transform.projection(big["x"], big["offsets"], big["w"], big["a"], big["b"], big["bias"], big["scale"], big["slots"], ctx=c)
                transform.projection_grad(big["x"], big["offsets"], big["w"], big["a"], big["b"], big["dy"], big["scale"], big["slots"], ctx=c)
                torch.cuda.synchronize()
                ref.check(host(y), *ref.projection("bfloat16", hb["x"], hb["offsets"], hb["w"], hb["a"], hb["b"], hb["bias"], hb["scale"], hb["slots"], hb["y0"]))
            everything(*eager)
            torch.cuda.synchronize()
            assert torch.equal(out["y"], eager[0]) and torch.equal(out["p"], eager[1]), turn
            for got, want in ((ga, eager[2]), (gp, eager[3])):
                for k in want:
                    assert torch.equal(got[k], want[k]), (turn, k)
    c.use_stream(None)
    del graph, fresh
    c.close()


def far_rows():
    """Rows whose elements lie past 2^31, and bytes past 2^32."""
    F, wide, I, O = 1100000, 2048, 72, 40
    room = torch.empty(F, wide, device="cuda", dtype=torch.bfloat16)
    x = room[:, wide - I:]
    x.copy_(torch.randn(F, I, device="cuda"))
    t, h = up(ref.make(10, (8, I, O, 3, 3, 8), slots=False), "bfloat16")
    off = torch.tensor([5, F // 2, F - 700, F - 3], device="cuda")
    y = torch.full((F, O), 3.0, device="cuda", dtype=torch.bfloat16)
    torch.cuda.synchronize()
    transform.affine(x, off, t["w3"], t["bias2"], out=y)
    p = transform.projection(x, off, t["w"], t["a"], t["b"], t["bias"], t["scale"])
    torch.cuda.synchronize()
    for lo, hi, k in ((5, 300, 0), (F - 2000, F - 700, 1), (F - 700, F - 3, 2)):
        xs, o = host(x[lo:hi]), np.array([0, hi - lo])
        zero = np.zeros((hi - lo, O))
        ref.check(host(y[lo:hi]), *ref.affine("bfloat16", xs, o, h["w3"][k:k + 1], h["bias2"][k:k + 1], None, zero), "affine")
        ref.check(host(p[lo:hi]), *ref.projection("bfloat16", xs, o, h["w"], h["a"][k:k + 1], h["b"][k:k + 1], h["bias"], h["scale"][k:k + 1], None, zero), "projection")
    assert bool((y[:5] == 3.0).all()) and bool((y[F - 3:] == 3.0).all())
    dy = torch.zeros(F, O, device="cuda", dtype=torch.bfloat16)
    dy[F - 600:F - 500] = torch.randn(100, O, device="cuda").to(torch.bfloat16)
    torch.cuda.synchronize()
    g = transform.affine_grad(x, off, t["w3"], dy, want=("w", "bias"))
    torch.cuda.synchronize()
    want = host(dy[F - 600:F - 500]).T @ host(x[F - 600:F - 500])
    size = np.abs(host(dy[F - 600:F - 500])).T @ np.abs(host(x[F - 600:F - 500]))
    ref.check(host(g["w"][2]), want, ref.rounded("bfloat16", want, 104 * 2.0 ** -24 * size))          # the zeros add nothing
    assert not bool(g["w"][:2].any())


def unchosen_streams():
    """No stream was chosen: a call waits for what its tensors come from, and is done when it returns."""
    c = _ffi.Context(0)
    t, h = up(ref.make(30, (4000, 64, 48, 5, 5, 8), slots=False), "float32")
    want, bound = ref.affine("float32", h["x"], h["offsets"], h["w3"], h["bias2"], None, h["y0"])
    slow = torch.randn(4096, 4096, device="cuda")
    for s in (torch.cuda.Stream(), torch.cuda.default_stream()):
        late = torch.zeros_like(t["x"])
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            for _ in range(20):
                slow = slow @ slow * 1e-3
            late.copy_(t["x"])
        y = transform.affine(late, t["offsets"], t["w3"], t["bias2"], ctx=c)
        z = y + 0
        torch.cuda.synchronize()
        ref.check(host(z), want, bound)
    c.close()


def pinned():
    """Pinned host arrays may change as soon as the call is back."""
    s = torch.cuda.Stream()
    c = _ffi.Context(0)
    c.use_stream(s)
    t, h = up(ref.make(31, (300, 512, 512, 40, 40, 8), slots=False), "float32")
    want, bound = ref.affine("float32", h["x"], h["offsets"], h["w3"], None, None, h["y0"])
    w = torch.empty(t["w3"].shape, pin_memory=True)
    w.copy_(t["w3"])
    off = torch.empty(t["offsets"].shape, dtype=torch.int64, pin_memory=True)
    off.copy_(t["offsets"])
    slow = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        for _ in range(20):
            slow = slow @ slow * 1e-3
        y = transform.affine(t["x"], off.numpy(), w.numpy(), ctx=c)
    w.fill_(float("nan"))
    off.fill_(0)
    torch.cuda.synchronize()
    ref.check(host(y), want, bound)
    c.use_stream(None)
    c.close()


def graph_outlives_context():
    """Captured while the context profiles; replayed after it was closed, on workspaces that stay."""
    s = torch.cuda.Stream()
    c = _ffi.Context(0)
    c.use_stream(s)
    t, h = up(ref.make(32, (500, 72, 80, 4, 3, 16)), "float32")
    y = torch.zeros_like(t["y0"])
    run = lambda: transform.projection(t["x"], t["offsets"], t["w"], t["a"], t["b"], t["bias"], t["scale"], t["slots"], out=y, ctx=c)
    with torch.cuda.stream(s):
        run()
        torch.cuda.synchronize()
        c.prof_enable(True)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            run()
        run()
        torch.cuda.synchronize()
        assert [v[0] for k, v in c.prof_report().items() if k.startswith("projection")] == [1, 1]      # the eager call's
        c.prof_enable(False)
        c.use_stream(None)
        c.close()
        other = [torch.full((1 << 20,), float("nan"), device="cuda") for _ in range(4)]
        want, bound = ref.projection("float32", h["x"], h["offsets"], h["w"], h["a"], h["b"], h["bias"], h["scale"], h["slots"], h["y0"])
        for _ in range(3):
            y.fill_(5.0)
            graph.replay()
            torch.cuda.synchronize()
            ref.check(host(y), want, bound)
        del other


CHECKS = {f.__name__: f for f in (bfloat16, bfloat16_wide, strides, streams, graphs, far_rows, unchosen_streams, pinned, graph_outlives_context)}

if __name__ == "__main__":
    for name in sys.argv[1:]:
        print("begin", name, flush=True)
        try:
            CHECKS[name]()
            print("RESULT", name, "ok", flush=True)
        except Exception:
            traceback.print_exc()
            print("RESULT", name, "failed", flush=True)
            if "HIP error" in traceback.format_exc():
                break                                                      # nothing more on a GPU that reports an error
