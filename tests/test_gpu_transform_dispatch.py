"""GPU: batches whose mean says little about their segments -- one long segment beside thousands of short or empty ones: every form
that may be chosen for them, and no cliff in time."""
import numpy as np
import pytest

import _transform_ref as ref
from test_gpu_transform_limits import check_columns

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from lnasr import _ffi
    c = _ffi.Context(0)
    yield c
    c.close()


def skewed(rng, kind, short, count, long, I, O, G=5):
    sizes = np.full(count, short, dtype=np.int64)
    sizes[count // 2] = long
    off = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int64)
    F = int(off[-1])
    return (rng.standard_normal((F, I)).astype(kind), off, (rng.standard_normal((G, O, I)) / np.sqrt(I)).astype(kind),
            rng.integers(0, G, count).astype(np.int32))


@pytest.mark.parametrize("kind", ["float64", "float32", "float16"])
@pytest.mark.parametrize("short,count,long", [(1, 3000, 9000), (0, 5000, 6000), (3, 800, 40), (20, 300, 3000), (70, 40, 5000)], ids=str)
def test_long_segments_among_short_ones(ctx, kind, short, count, long):
    rng = np.random.default_rng(8)
    for I, O in ((130, 264), (72, 40)):
        x, off, w, sl = skewed(rng, kind, short, count, long, I, O)
        y = ctx.affine(ctx.to_device(x), off, ctx.to_device(w), slots=sl).to_host()
        rows = np.repeat(sl, np.diff(off))
        check_columns(kind, x, y, w, rows, "y")
        wt = np.ascontiguousarray(w.transpose(0, 2, 1))
        g = ctx.affine_grad(ctx.to_device(np.ones((len(x), O), kind)), off, ctx.to_device(wt), ctx.to_device(x), sl, want=("x",))["x"].to_host()
        check_columns(kind, x, g, w, rows, "dx")


def test_a_long_segment_costs_what_it_costs_alone(ctx):
    """100,000 rows beside 10,000 empty segments: blocks of 16 rows, as their mean of ten suggests, took 22 times as long as without
    the empty ones; the tiles take four to five, most of it to find that there is nothing to do."""
    import time
    rng = np.random.default_rng(9)
    F, I, O, S = 100000, 1024, 1024, 10001
    x, w = ctx.to_device(rng.standard_normal((F, I)).astype(np.float16)), ctx.to_device((rng.standard_normal((1, O, I)) / 32).astype(np.float16))
    y = ctx.to_device(np.zeros((F, O), np.float16))
    sizes = np.zeros(S, dtype=np.int64)
    sizes[S // 2] = F
    many = ctx.to_device(np.concatenate([[0], np.cumsum(sizes)]).astype(np.int64))
    one, slots = ctx.to_device(np.array([0, F], dtype=np.int64)), ctx.to_device(np.zeros(S, dtype=np.int32))

    def best(*args, **kw):
        times = []
        for _ in range(5):
            ctx.sync()
            t = time.perf_counter()
            for _ in range(10):
                ctx.affine(x, *args, out=y, **kw)
            ctx.sync()
            times.append(time.perf_counter() - t)
        return min(times)

    ratio = best(many, w, slots=slots) / best(one, w)
    print("ratio %.1f" % ratio)
    assert ratio < 10


@pytest.mark.parametrize("size,slots", [((33000, 520, 1030, 30, 9, 8), True), ((33000, 1030, 520, 120, 9, 8), True), ((33000, 513, 1024, 90, 90, 8), False)],
                         ids=str)
def test_largest_sums(ctx, size, slots):
    """256 x 256 sums over sorted segments, over segments as they lie, over the batch as one: groups without rows, uneven edges, short
    last steps."""
    d = ref.make(75, size, slots=slots)
    d = {k: v if v is None or k in ("offsets", "slots", "scale") else v.astype(np.float16) for k, v in d.items()}
    got = ctx.affine_grad(d["x"], d["offsets"], d["w3"], d["dy"], d["slots"], want=("w", "bias"))
    want, err = ref.affine_grad("float16", d["x"], d["offsets"], d["w3"], d["dy"], d["slots"], d["dx0"])
    for k in got:
        ref.check(got[k], want[k], err[k], "affine_grad " + k)
    got = ctx.projection_grad(d["x"], d["offsets"], d["w"], d["a"], d["b"], d["dy"], d["scale"], d["slots"], want=("w", "bias", "a"))
    want, err = ref.projection_grad("float16", d["x"], d["offsets"], d["w"], d["a"], d["b"], d["dy"], d["scale"], d["slots"], d["dx0"])
    for k in got:
        ref.check(got[k], want[k], err[k], "projection_grad " + k)
