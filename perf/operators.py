"""What is measured of the feature transforms: cases, their inputs, a plain form of each operator, and its exact value.

Two operators of `lnasr.transform`, each with its gradient:

  affine      y[r] = W[k] x[r] + c[k]                             W [G, dout, din], c [G, dout]
              an affine transform per speaker, class or expert; rows come in segments (utterances), segment s holds rows
              offsets[s] .. offsets[s+1] and names its transform k = slots[s] (no slots: k = s)
  projection  y[r] = W x[r] + c + scale[k] * B[k] (A[k] x[r])     W [dout, din], A [G, rank, din], B [G, dout, rank]
              one projection that all rows share, beside it a low-rank adapter per speaker or request; slot -1: none

`run` with own = False computes them from elementary torch operations in 32 bits (64 for float64 inputs), rounded once.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

TYPES = {"f64": torch.float64, "f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f64": 8, "f32": 4, "f16": 2, "bf16": 2}


def _case(name, op, dtype, rows, din, dout, segments, groups, rank=0, grad=False, ones=False, slots=True, shared=False):
    """rows: all rows of the batch.  ones: every segment is a single row.  slots: segments name their group (several may
    name the same one), otherwise segment s is group s.  shared: the gradient of the shared W and c of a projection is asked
    for too."""
    c = {"op": op, "dtype": dtype, "rows": rows, "din": din, "dout": dout, "segments": segments, "groups": groups,
         "rank": rank, "grad": grad, "ones": ones, "slots": slots, "shared": shared}
    return {"name": name, **c} if name else c


def listed():
    return [
        # live audio: the newest MFCC frame of 64 speakers, each with a transform of their own
        _case("affine-live", "affine", "f64", 64, 39, 39, 64, 64, ones=True, slots=False),
        # a decoding batch: 1024 utterances of 256 speakers, 1,024,000 MFCC frames, before the GMM bank scores them
        _case("affine-batch", "affine", "f64", 1024000, 39, 39, 1024, 256),
        # nine spliced frames per row (9 x 39) to 40 dimensions, one discriminant transform per class; odd sizes
        _case("affine-splice", "affine", "f32", 200003, 351, 40, 77, 12),
        # experts' products of a wide layer: 32 experts, ragged shares of 65,536 rows
        _case("affine-experts", "affine", "bf16", 65536, 2048, 2048, 32, 32, slots=False),
        # estimating the speakers' transforms: gradients of features, matrices and offsets
        _case("affine-batch-grad", "affine", "f64", 300007, 39, 39, 300, 64, grad=True),
        # training the experts
        _case("affine-experts-grad", "affine", "bf16", 32768, 1024, 2048, 16, 16, grad=True, slots=False),
        # serving: one row from each of 64 requests, each with its adapter
        _case("projection-live", "projection", "bf16", 64, 2048, 2048, 64, 48, rank=16, ones=True),
        # serving: prompts of 24 requests, ragged
        _case("projection-prompts", "projection", "f16", 16384, 1024, 2048, 24, 16, rank=32),
        # spliced features of a test set through a shared projection with speakers' adapters; odd sizes
        _case("projection-splice", "projection", "f32", 120011, 351, 128, 190, 40, rank=8),
        # training the adapters, the shared matrix frozen
        _case("projection-adapt", "projection", "bf16", 16384, 1024, 1024, 20, 12, rank=16, grad=True),
        # training matrix and adapters together
        _case("projection-train", "projection", "f32", 20011, 429, 512, 33, 10, rank=8, grad=True, shared=True),
    ]


def draw(rng):
    def spread(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["affine", "projection"])
    dtype = rng.choice(["f64", "f32", "f16", "bf16"])
    grad = rng.random() < 0.4
    rank = spread(1, 64) if op == "projection" else 0
    wide = {"f64": 512, "f32": 1024, "f16": 2048, "bf16": 2048}[dtype]
    din, dout = spread(5, wide), spread(5, wide)
    if rng.random() < 0.5:                                 # widths as they are usually chosen
        din, dout = (-(-v // 8) * 8 if v > 16 else v for v in (din, dout))
    most = {"f64": 8e9, "f32": 3e10, "f16": 3e11, "bf16": 3e11}[dtype] / (3 if grad else 1)
    rows = spread(1, 1000000)
    rows = int(max(1, min(rows, most / (2.0 * din * dout), 3e8 / ((din + dout) * 8.0))))
    ones = rows <= 2048 and rng.random() < 0.4
    per = din * dout if op == "affine" else rank * (din + dout)
    few = max(1, int(min(1024, 2.5e8 / per)))              # the matrices of all segments stay in reach
    if ones:
        rows = min(rows, few)
    segments = rows if ones else spread(1, max(1, min(rows, few)))
    slots = rng.random() < 0.7
    groups = spread(1, segments) if slots else segments
    return _case(None, op, dtype, rows, din, dout, segments, groups, rank=rank, grad=grad, ones=ones, slots=slots,
                 shared=op == "projection" and grad and rng.random() < 0.5)


def work(case):
    """Each input read once, each output written once; two operations to a product."""
    F, I, O, G, R = (case[k] for k in ("rows", "din", "dout", "groups", "rank"))
    used = min(G, case["segments"])
    e = BYTES[case["dtype"]]
    if case["op"] == "affine":
        mats = used * O * (I + 1)
        if not case["grad"]:
            return {"bytes": e * (F * (I + O) + mats), "flops": 2.0 * F * I * O}
        return {"bytes": e * (F * (2 * I + O) + used * O * I + G * O * (I + 1)), "flops": 4.0 * F * I * O}
    low = used * R * (I + O)
    if not case["grad"]:
        return {"bytes": e * (F * (I + O) + O * (I + 1) + low), "flops": 2.0 * F * (I * O + R * (I + O))}
    out = G * R * (I + O) + (O * (I + 1) if case["shared"] else 0)
    flops = 2.0 * F * (I * O * (2 if case["shared"] else 1) + R * (3 * I + 2 * O))
    return {"bytes": e * (F * (2 * I + O) + O * I + low + out), "flops": flops}


def prepare(case, seed):
    F, I, O, S, G, R = (case[k] for k in ("rows", "din", "dout", "segments", "groups", "rank"))
    t = TYPES[case["dtype"]]
    host = np.random.RandomState(seed % (2 ** 31))
    if case["ones"]:
        sizes = np.ones(S, dtype=np.int64)
    else:                                                  # utterance lengths spread about their mean; some may be empty
        share = host.lognormal(0.0, 0.6, S)
        cuts = np.floor(np.cumsum(share) / share.sum() * F + 0.5).astype(np.int64)
        cuts[-1] = F
        sizes = np.diff(np.concatenate([[0], cuts]))
    offsets = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int64)
    slots = None
    if case["slots"]:
        slots = host.randint(0, G, S).astype(np.int32)
        if case["op"] == "projection" and S > 4:
            slots[host.randint(0, S, S // 8 + 1)] = -1     # requests without an adapter
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, size=1.0):
        # drawn in 32 bits and rounded: the same work whatever the type
        return (torch.randn(*shape, generator=g, device="cuda") * size).to(t)

    s = {"op": case["op"], "grad": case["grad"], "shared": case["shared"], "longest": int(sizes.max()),
         "x": normal(F, I), "offsets": torch.from_numpy(offsets).cuda(),
         "slots": None if slots is None else torch.from_numpy(slots).cuda()}
    out = {"y": torch.zeros(F, O, dtype=t, device="cuda")}
    if case["op"] == "affine":
        s["w"], s["bias"] = normal(G, O, I, size=I ** -0.5), normal(G, O, size=0.1)
        if case["grad"]:
            out = {"x": torch.empty_like(s["x"]), "w": torch.empty_like(s["w"]), "bias": torch.empty_like(s["bias"])}
    else:
        s["w"], s["bias"] = normal(O, I, size=I ** -0.5), normal(O, size=0.1)
        s["a"], s["b"] = normal(G, R, I, size=I ** -0.5), normal(G, O, R, size=0.3 * R ** -0.5)
        s["scale"] = torch.from_numpy(host.uniform(0.5, 2.0, G)).cuda()
        if case["grad"]:
            out = {k: torch.empty_like(s[k]) for k in (("x", "a", "b", "w", "bias") if case["shared"] else ("x", "a", "b"))}
    if case["grad"]:
        s["dy"] = normal(F, O, size=0.05)
    s["out"] = out                                         # where the framework writes its answer
    return s


# ---- the framework's operators ---------------------------------------------------------------------------------------
def _framework():
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ln-asr_amd")
    root = here if os.path.isdir(here) else os.path.join(os.getcwd(), "ln-asr_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from lnasr import transform
    return transform


def _run_own(s):
    tr = _framework()
    ctx = tr.default_ctx()
    ctx.use_stream(torch.cuda.current_stream().cuda_stream)
    out = s["out"]
    if s["op"] == "affine":
        if s["grad"]:
            return tr.affine_grad(s["x"], s["offsets"], s["w"], s["dy"], slots=s["slots"], out=out)
        return tr.affine(s["x"], s["offsets"], s["w"], s["bias"], slots=s["slots"], out=out["y"])
    if s["grad"]:
        return tr.projection_grad(s["x"], s["offsets"], s["w"], s["a"], s["b"], s["dy"], scale=s["scale"], slots=s["slots"],
                                  out=out)
    return tr.projection(s["x"], s["offsets"], s["w"], s["a"], s["b"], bias=s["bias"], scale=s["scale"], slots=s["slots"],
                         out=out["y"])


# ---- the plain form --------------------------------------------------------------------------------------------------
def _run_plain(s):
    t = s["x"].dtype
    f = torch.float64 if t == torch.float64 else torch.float32
    F, S, L = s["x"].shape[0], s["offsets"].shape[0] - 1, s["longest"]
    rows = torch.arange(F, device="cuda")
    seg = torch.searchsorted(s["offsets"], rows, right=True) - 1
    pos = rows - s["offsets"][seg]
    slot = torch.arange(S, device="cuda") if s["slots"] is None else s["slots"].long()
    has = slot >= 0
    slot = slot.clamp(min=0)

    def padded(v):                                         # [F, D] -> [S, L, D], zeros behind each segment's last row
        p = torch.zeros(S, L, v.shape[1], dtype=f, device="cuda")
        p[seg, pos] = v
        return p

    def joined(v):                                         # [S, ...] -> [G, ...]: the segments of a group summed
        G = s["w"].shape[0] if s["op"] == "affine" else s["a"].shape[0]
        return torch.zeros((G,) + v.shape[1:], dtype=f, device="cuda").index_add_(0, slot, v)

    x = s["x"].to(f)
    if s["op"] == "affine":
        w = s["w"][slot].to(f)
        if not s["grad"]:
            y = torch.bmm(padded(x), w.transpose(1, 2).contiguous()) + s["bias"][slot].to(f)[:, None]
            return y[seg, pos].to(t)
        dy = padded(s["dy"].to(f))
        dw = torch.bmm(dy.transpose(1, 2).contiguous(), padded(x))
        return {"x": torch.bmm(dy, w)[seg, pos].to(t), "w": joined(dw).to(t), "bias": joined(dy.sum(1)).to(t)}
    w = s["w"].to(f)
    a, b = s["a"][slot].to(f), s["b"][slot].to(f)
    scale = (s["scale"][slot] * has).to(f)[:, None, None]
    px = padded(x)
    low = torch.bmm(px, a.transpose(1, 2).contiguous()) * scale
    if not s["grad"]:
        y = x @ w.t() + s["bias"].to(f) + torch.bmm(low, b.transpose(1, 2).contiguous())[seg, pos]
        return y.to(t)
    dy = s["dy"].to(f)
    pdy = padded(dy)
    dlow = torch.bmm(pdy, b) * scale
    got = {"x": (dy @ w + torch.bmm(dlow, a)[seg, pos]).to(t),
           "a": joined(torch.bmm(dlow.transpose(1, 2).contiguous(), px)).to(t),
           "b": joined(torch.bmm(pdy.transpose(1, 2).contiguous(), low)).to(t)}
    if s["shared"]:
        got["w"], got["bias"] = (dy.t() @ x).to(t), dy.sum(0).to(t)
    return got


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the exact value, segment by segment in 64 bits ------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in s.items()}
    x, w, cuts = d["x"], d["w"], s["offsets"].tolist()
    names = list(range(len(cuts) - 1)) if s["slots"] is None else s["slots"].tolist()
    spans = [(k, slice(lo, hi)) for k, lo, hi in zip(names, cuts[:-1], cuts[1:]) if hi > lo]
    zero = {k: torch.zeros(v.shape, dtype=torch.float64, device="cuda") for k, v in s["out"].items()}
    if case["op"] == "affine":
        for k, r in spans:
            if not case["grad"]:
                zero["y"][r] = torch.mm(x[r], w[k].t()).add_(d["bias"][k])
                continue
            dy = d["dy"][r]
            zero["x"][r] = dy.mm(w[k])
            zero["w"][k] += dy.t().mm(x[r])
            zero["bias"][k] += dy.sum(dim=0)
        return zero if case["grad"] else zero["y"]
    if not case["grad"]:
        zero["y"] = torch.addmm(d["bias"], x, w.t())
    else:
        zero["x"] = d["dy"].mm(w)
        if case["shared"]:
            zero["w"], zero["bias"] = d["dy"].t().mm(x), d["dy"].sum(dim=0)
    for k, r in spans:
        if k < 0:
            continue
        A, B, c = d["a"][k], d["b"][k], d["scale"][k]
        if not case["grad"]:
            zero["y"][r] += c * x[r].mm(A.t()).mm(B.t())
            continue
        dy = d["dy"][r]
        dp = c * dy.mm(B)
        zero["x"][r] += dp.mm(A)
        zero["a"][k] += dp.t().mm(x[r])
        zero["b"][k] += c * dy.t().mm(x[r].mm(A.t()))
    return zero if case["grad"] else zero["y"]
