"""Plain 64-bit forms of the feature transforms, segment by segment, with the error each result may have.

An error bound counts roundings.  A sum of n products held in a type of unit roundoff u (2^-24; 2^-53 for float64) is off by at
most (n + 2) u sum |products|, in whatever order it runs; the result is then rounded once to its type (half a step, h = eps / 2
of that type, or half a step among its subnormals).  The middle of a projection is rounded to the type as well, and that
error is carried through the second product.  The reference's own sums (64 bits) err by as much again for float64: both count."""
import numpy as np

STEP = {"float64": 2.0 ** -53, "float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TINY = {"float64": 2.0 ** -1075, "float32": 2.0 ** -150, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -134}


def unit(kind):
    return 2.0 ** -52 if kind == "float64" else 2.0 ** -24            # float64: the reference's roundings too


def rounded(kind, value, err):
    return err + STEP[kind] * (np.abs(value) + err) + TINY[kind]


def spans(offsets, slots):
    for s in range(len(offsets) - 1):
        lo, hi = int(offsets[s]), int(offsets[s + 1])
        if hi > lo:
            yield (s if slots is None else int(slots[s])), slice(lo, hi)


def affine(kind, x, offsets, w, bias, slots, before):
    """(y, bound): rows of no segment keep `before`, exactly."""
    x, w = x.astype(np.float64), w.astype(np.float64)
    y, err = before.astype(np.float64).copy(), np.zeros(before.shape)
    u, n = unit(kind), x.shape[1] + 4
    for k, r in spans(offsets, slots):
        b = 0.0 if bias is None else bias[k].astype(np.float64)
        y[r] = x[r] @ w[k].T + b
        err[r] = rounded(kind, y[r], n * u * (np.abs(x[r]) @ np.abs(w[k]).T + np.abs(b)))
    return y, err


def affine_grad(kind, x, offsets, w, dy, slots, before):
    x, w, dy = x.astype(np.float64), w.astype(np.float64), dy.astype(np.float64)
    g = {"x": before.astype(np.float64).copy(), "w": np.zeros(w.shape), "bias": np.zeros(w.shape[:2])}
    size = {k: np.zeros(v.shape) for k, v in g.items()}
    rows = np.zeros(w.shape[0])
    err = {"x": np.zeros(before.shape)}
    u = unit(kind)
    for k, r in spans(offsets, slots):
        g["x"][r] = dy[r] @ w[k]
        err["x"][r] = rounded(kind, g["x"][r], (w.shape[1] + 4) * u * (np.abs(dy[r]) @ np.abs(w[k])))
        g["w"][k] += dy[r].T @ x[r]
        size["w"][k] += np.abs(dy[r]).T @ np.abs(x[r])
        g["bias"][k] += dy[r].sum(0)
        size["bias"][k] += np.abs(dy[r]).sum(0)
        rows[k] += r.stop - r.start
    err["w"] = rounded(kind, g["w"], (rows[:, None, None] + 4) * u * size["w"])
    err["bias"] = rounded(kind, g["bias"], (rows[:, None] + 4) * u * size["bias"])
    return g, err


def _middle(kind, v, m, c):
    """c * v m^T as the kernels hold it: its value, and how far the held one may be off."""
    p = c * (v @ m.T)
    return p, rounded(kind, p, (v.shape[1] + 4) * unit(kind) * abs(c) * (np.abs(v) @ np.abs(m).T))


def projection(kind, x, offsets, w, a, b, bias, scale, slots, before):
    x, w, a, b = (t.astype(np.float64) for t in (x, w, a, b))
    y, err = before.astype(np.float64).copy(), np.zeros(before.shape)
    u, n = unit(kind), x.shape[1] + a.shape[1] + 8
    c0 = 0.0 if bias is None else bias.astype(np.float64)
    for k, r in spans(offsets, slots):
        y[r] = x[r] @ w.T + c0
        size, e = np.abs(x[r]) @ np.abs(w).T + np.abs(c0), 0.0
        if k >= 0:
            p, ep = _middle(kind, x[r], a[k], 1.0 if scale is None else scale[k])
            y[r] += p @ b[k].T
            size = size + (np.abs(p) + ep) @ np.abs(b[k]).T
            e = ep @ np.abs(b[k]).T
        err[r] = rounded(kind, y[r], n * u * size + e)
    return y, err


def projection_grad(kind, x, offsets, w, a, b, dy, scale, slots, before):
    x, w, a, b, dy = (t.astype(np.float64) for t in (x, w, a, b, dy))
    g = {"x": before.astype(np.float64).copy(), "a": np.zeros(a.shape), "b": np.zeros(b.shape), "w": np.zeros(w.shape),
         "bias": np.zeros(w.shape[0])}
    size = {k: np.zeros(v.shape) for k, v in g.items()}
    more = {k: np.zeros(v.shape) for k, v in g.items()}
    rows = np.zeros(a.shape[0])
    u, all_rows = unit(kind), 0
    for k, r in spans(offsets, slots):
        g["x"][r] = dy[r] @ w
        size["x"][r] = np.abs(dy[r]) @ np.abs(w)
        g["w"] += dy[r].T @ x[r]
        size["w"] += np.abs(dy[r]).T @ np.abs(x[r])
        g["bias"] += dy[r].sum(0)
        size["bias"] += np.abs(dy[r]).sum(0)
        all_rows += r.stop - r.start
        if k < 0:
            continue
        c = 1.0 if scale is None else scale[k]
        d, ed = _middle(kind, dy[r], b[k].T, c)
        p, ep = _middle(kind, x[r], a[k], c)
        g["x"][r] += d @ a[k]
        size["x"][r] += (np.abs(d) + ed) @ np.abs(a[k])
        more["x"][r] = ed @ np.abs(a[k])
        g["a"][k] += d.T @ x[r]
        size["a"][k] += (np.abs(d) + ed).T @ np.abs(x[r])
        more["a"][k] += ed.T @ np.abs(x[r])
        g["b"][k] += dy[r].T @ p
        size["b"][k] += np.abs(dy[r]).T @ (np.abs(p) + ep)
        more["b"][k] += np.abs(dy[r]).T @ ep
        rows[k] += r.stop - r.start
    n = {"x": w.shape[0] + a.shape[1] + 8, "a": rows[:, None, None] + 4, "b": rows[:, None, None] + 4, "w": all_rows + 4, "bias": all_rows + 4}
    err = {k: rounded(kind, g[k], n[k] * u * size[k] + more[k]) for k in g}
    out = np.ones(before.shape[0], dtype=bool)
    for _, r in spans(offsets, slots):
        out[r] = False
    err["x"][out] = 0.0                                                # rows of no segment: as they were
    return g, err


def check(got, want, bound, what=""):
    got, want = np.asarray(got, dtype=np.float64), np.asarray(want)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~(np.abs(got - want) <= bound)
    if bad.any():
        i = tuple(np.argwhere(bad)[0])
        raise AssertionError("%s: %d of %d off, first at %s: %r for %r, may be off by %g" % (
            what, bad.sum(), bad.size, i, got[i], want[i], bound[i]))


# rows, din, dout, segments, groups, rank: one row; odd widths; widths and heights on and about the tile edges; long segments; many
# single rows; empty segments; more groups than segments
SIZES = [(1, 1, 1, 1, 1, 1), (1, 39, 39, 1, 3, 2), (5, 7, 3, 2, 2, 3), (64, 39, 39, 64, 64, 4), (300, 39, 40, 7, 3, 8),
         (129, 16, 16, 3, 2, 16), (2000, 39, 39, 2, 2, 5), (513, 63, 65, 9, 4, 17), (700, 64, 64, 5, 9, 8), (333, 351, 40, 6, 3, 8),
         (17, 128, 129, 17, 5, 33), (200, 130, 256, 4, 4, 64), (90, 512, 96, 40, 7, 1), (70, 65, 513, 3, 2, 70), (4097, 48, 24, 11, 3, 4),
         (640, 256, 320, 5, 3, 16), (31, 1024, 264, 31, 4, 24), (1500, 392, 136, 3, 3, 32)]


def make(seed, size, empties=True, slots=True, single=False, negative=False):
    """Inputs in float64 (values that float16 and bfloat16 hold exactly after their own rounding by the caller)."""
    F, I, O, S, G, R = size
    rng = np.random.default_rng(seed)
    if single:
        S = F
        offsets = np.arange(F + 1)
    else:
        cuts = np.sort(rng.integers(0, F + 1, S - 1))
        if empties and S > 2:
            cuts[S // 2] = cuts[S // 2 - 1]                            # an empty segment
        offsets = np.concatenate([[0], np.sort(cuts), [F]])
    if not slots:
        G = S
    sl = rng.integers(-1 if negative else 0, G, S).astype(np.int32) if slots else None
    d = {"x": rng.standard_normal((F, I)), "offsets": offsets.astype(np.int64), "slots": sl, "dy": rng.standard_normal((F, O)),
         "w3": rng.standard_normal((G, O, I)) / np.sqrt(I), "bias2": rng.standard_normal((G, O)), "w": rng.standard_normal((O, I)) / np.sqrt(I),
         "bias": rng.standard_normal(O), "a": rng.standard_normal((G, R, I)) / np.sqrt(I), "b": rng.standard_normal((G, O, R)) / np.sqrt(R),
         "scale": rng.uniform(0.5, 2.0, G), "y0": rng.standard_normal((F, O)), "dx0": rng.standard_normal((F, I))}
    return d
