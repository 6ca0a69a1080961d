"""GPU: a projection's narrow middle, scale A x and in the gradients scale B^T dy, is held in 32 bits beside 16-bit features: the
results' bounds have one rounding to 16 bits, their own, and the middle's range is not that of the features."""
import numpy as np
import pytest

import _transform_ref as ref
from _transform_bf16 import Calls

pytestmark = pytest.mark.gpu

KINDS = ["float16", "bfloat16"]
# rows, din, dout, segments, groups, rank: the forms for few rows, tiles of either width, the largest tiles; ranks of several steps
WIDE = [(2000, 130, 200, 6, 3, 16), (2000, 200, 130, 160, 9, 40), (300, 24, 40, 5, 3, 300), (9001, 840, 2056, 5, 4, 24), (16500, 1030, 270, 9, 3, 9),
        (24000, 512, 520, 40, 32, 33), (20000, 48, 40, 30, 8, 8), (6000, 40, 24, 30, 8, 64), (30000, 1024, 1030, 12, 5, 8)]


@pytest.fixture(scope="module")
def ctx():
    from lnasr import _ffi
    c = _ffi.Context(0)
    yield c
    c.close()


@pytest.fixture(autouse=True)
def middle_in_32_bits(monkeypatch):
    plain = ref._middle
    monkeypatch.setattr(ref, "_middle", lambda kind, v, m, c: plain("float32", v, m, c))


def inputs(calls, seed, size, **kw):
    d = ref.make(seed, size, **kw)
    return {k: v if v is None or k in ("offsets", "slots", "scale") else calls.round(v) for k, v in d.items()}


def both(ctx, kind, d):
    c = Calls(ctx, kind)
    y = c.projection(d)
    ref.check(y, *ref.projection(kind, d["x"], d["offsets"], d["w"], d["a"], d["b"], d["bias"], d["scale"], d["slots"], d["y0"]), "y")
    got = c.projection_grad(d)
    want, err = ref.projection_grad(kind, d["x"], d["offsets"], d["w"], d["a"], d["b"], d["dy"], d["scale"], d["slots"], d["dx0"])
    for k in want:
        ref.check(got[k], want[k], err[k], k)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", ref.SIZES, ids=str)
def test_bounds(ctx, kind, size):
    for seed, kw in ((1, {"negative": True}), (2, {"slots": False}), (3, {"single": True, "negative": True})):
        both(ctx, kind, inputs(Calls(ctx, kind), seed, size, **kw))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", WIDE, ids=str)
def test_bounds_of_wide_products(ctx, kind, size):
    both(ctx, kind, inputs(Calls(ctx, kind), 4, size, negative=True))


@pytest.mark.parametrize("size", [(40, 33, 40, 5, 3, 5), (700, 256, 320, 3, 2, 16), (16640, 1024, 1024, 2, 2, 16)], ids=str)
def test_range(ctx, size):
    """float16 features whose middle is past the type's largest value, or among its subnormals: results (of the adapters alone, W is
    zero) that are in its range are right."""
    c = Calls(ctx, "float16")
    d = inputs(c, 5, size)
    d["w"], d["bias"] = np.zeros_like(d["w"]), np.zeros_like(d["bias"])
    for up, down in ((2.0 ** 17, 2.0 ** -12), (2.0 ** -20, 2.0 ** 8)):
        for other, names in (("b", ("x", "a")), ("a", ("x", "b"))):
            e = dict(d, scale=d["scale"] * up)
            e[other] = c.round(d[other] * down)
            e["dy"] = c.round(d["dy"] * 2.0 ** -4)
            y = c.projection(e)
            ref.check(y, *ref.projection("float16", e["x"], e["offsets"], e["w"], e["a"], e["b"], e["bias"], e["scale"], e["slots"], e["y0"]), "y")
            got = c.projection_grad(e)
            want, err = ref.projection_grad("float16", e["x"], e["offsets"], e["w"], e["a"], e["b"], e["dy"], e["scale"], e["slots"], e["dx0"])
            for k in names:
                assert np.abs(want[k]).max() < 6e4
                ref.check(got[k], want[k], err[k], k)


@pytest.mark.parametrize("kind", KINDS)
def test_infinities_and_nan(ctx, kind):
    """A row of infinities, an adapter of NaN or infinity: where their products go, as in 32-bit arithmetic, and nowhere else."""
    c = Calls(ctx, kind)
    d = inputs(c, 6, (600, 72, 80, 6, 3, 8))
    d["slots"] = np.array([0, 1, 2, 0, 1, -1], dtype=np.int32)
    d["offsets"] = np.arange(0, 601, 100).astype(np.int64)
    for name, value in (("x", np.inf), ("a", np.nan), ("b", np.inf), ("b", -np.inf)):
        e = dict(d, **{name: d[name].copy()})
        sick = np.zeros(600, dtype=bool)
        if name == "x":
            e["x"][130, 3] = value
            sick[130] = True
        else:
            e[name][1] = value
            sick[100:200] = sick[400:500] = True
        y = c.projection(e)
        with np.errstate(invalid="ignore"):
            full = ref.projection(kind, e["x"], e["offsets"], e["w"], e["a"], e["b"], e["bias"], e["scale"], e["slots"], e["y0"])[0]
        assert np.array_equal(np.isnan(y), np.isnan(full)) and np.array_equal(np.isinf(y), np.isinf(full)), (name, value)
        assert np.array_equal(np.sign(y[np.isinf(full)]), np.sign(full[np.isinf(full)])), (name, value)
        want, err = ref.projection(kind, d["x"], d["offsets"], d["w"], d["a"], d["b"], d["bias"], d["scale"], d["slots"], d["y0"])
        ref.check(y[~sick], want[~sick], err[~sick], name)
        assert not np.isfinite(full[sick]).all()
