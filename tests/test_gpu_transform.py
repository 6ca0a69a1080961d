"""GPU: feature transforms through the C-ABI with numpy arrays and DeviceArrays, against plain 64-bit forms (_transform_ref.py:
the bounds count roundings).  Tensors of another library, bfloat16, streams and graphs: test_gpu_transform_tensors.py."""
import numpy as np
import pytest

import _transform_ref as ref

pytestmark = pytest.mark.gpu

KINDS = ["float64", "float32", "float16"]


@pytest.fixture(scope="module")
def ctx():
    from lnasr import _ffi
    c = _ffi.Context(0)
    yield c
    c.close()


def typed(d, kind):
    return {k: v if k in ("offsets", "slots", "scale") else v.astype(kind) for k, v in d.items()}


def run_affine(ctx, kind, d, device):
    y = d["y0"].copy()
    up = ctx.to_device if device else (lambda v: v)
    args = [up(d["x"]), up(d["offsets"]), up(d["w3"]), up(d["bias2"])]
    out = ctx.to_device(y) if device else y
    got = ctx.affine(*args, slots=None if d["slots"] is None else up(d["slots"]), out=out)
    assert got is out
    got = got.to_host() if device else got
    ref.check(got, *ref.affine(kind, d["x"], d["offsets"], d["w3"], d["bias2"], d["slots"], d["y0"]), "y")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", ref.SIZES, ids=str)
def test_affine(ctx, kind, size):
    run_affine(ctx, kind, typed(ref.make(1, size), kind), device=False)
    run_affine(ctx, kind, typed(ref.make(2, size, slots=False), kind), device=True)
    run_affine(ctx, kind, typed(ref.make(3, size, single=True), kind), device=True)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", ref.SIZES, ids=str)
def test_affine_grad(ctx, kind, size):
    for seed, kw in ((1, {}), (2, {"slots": False}), (3, {"single": True})):
        d = typed(ref.make(seed, size, **kw), kind)
        out = {"x": d["dx0"].copy(), "w": np.full(d["w3"].shape, np.nan, kind), "bias": np.full(d["bias2"].shape, np.nan, kind)}
        got = ctx.affine_grad(d["x"], d["offsets"], d["w3"], d["dy"], slots=d["slots"], out=out)
        want, err = ref.affine_grad(kind, d["x"], d["offsets"], d["w3"], d["dy"], d["slots"], d["dx0"])
        for k in want:
            ref.check(got[k], want[k], err[k], k)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", ref.SIZES, ids=str)
def test_projection(ctx, kind, size):
    for seed, kw in ((1, {"negative": True}), (2, {"slots": False}), (3, {"single": True, "negative": True})):
        d = typed(ref.make(seed, size, **kw), kind)
        y = ctx.projection(d["x"], d["offsets"], d["w"], d["a"], d["b"], d["bias"], d["scale"], d["slots"], out=d["y0"].copy())
        ref.check(y, *ref.projection(kind, d["x"], d["offsets"], d["w"], d["a"], d["b"], d["bias"], d["scale"], d["slots"], d["y0"]), "y")
    y = ctx.projection(d["x"], d["offsets"], d["w"], d["a"], d["b"], slots=d["slots"])               # neither bias nor scale
    ref.check(y, *ref.projection(kind, d["x"], d["offsets"], d["w"], d["a"], d["b"], None, None, d["slots"], d["y0"]), "y")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", ref.SIZES, ids=str)
def test_projection_grad(ctx, kind, size):
    for seed, kw in ((1, {"negative": True}), (2, {"slots": False}), (3, {"single": True, "negative": True})):
        d = typed(ref.make(seed, size, **kw), kind)
        got = ctx.projection_grad(d["x"], d["offsets"], d["w"], d["a"], d["b"], d["dy"], d["scale"], d["slots"])
        want, err = ref.projection_grad(kind, d["x"], d["offsets"], d["w"], d["a"], d["b"], d["dy"], d["scale"], d["slots"], d["dx0"])
        assert sorted(got) == sorted(want)
        for k in want:
            ref.check(got[k], want[k], err[k], k)


@pytest.mark.parametrize("size", [(9001, 840, 2056, 5, 4, 24), (17000, 72, 1032, 3, 2, 40), (16500, 1030, 270, 9, 3, 9),
                                  (24000, 512, 520, 40, 32, 16)], ids=str)
def test_wide_tiles(ctx, size):
    """16-bit products wide and long enough for the largest tiles: k of several turns of the buffers, of one step and of less,
    uneven edges, segments that end inside a tile."""
    d = typed(ref.make(12, size, empties=False, negative=True), "float16")
    y = ctx.projection(d["x"], d["offsets"], d["w"], d["a"], d["b"], d["bias"], d["scale"], d["slots"])
    ref.check(y, *ref.projection("float16", d["x"], d["offsets"], d["w"], d["a"], d["b"], d["bias"], d["scale"], d["slots"], d["y0"]), "projection")
    got = ctx.projection_grad(d["x"], d["offsets"], d["w"], d["a"], d["b"], d["dy"], d["scale"], d["slots"])
    want, err = ref.projection_grad("float16", d["x"], d["offsets"], d["w"], d["a"], d["b"], d["dy"], d["scale"], d["slots"], d["dx0"])
    for k in want:
        ref.check(got[k], want[k], err[k], "projection_grad " + k)
    d["slots"] = np.maximum(d["slots"], 0)
    y = ctx.affine(d["x"], d["offsets"], d["w3"], d["bias2"], d["slots"])
    ref.check(y, *ref.affine("float16", d["x"], d["offsets"], d["w3"], d["bias2"], d["slots"], d["y0"]), "affine")
    got = ctx.affine_grad(d["x"], d["offsets"], d["w3"], d["dy"], d["slots"])
    want, err = ref.affine_grad("float16", d["x"], d["offsets"], d["w3"], d["dy"], d["slots"], d["dx0"])
    for k in want:
        ref.check(got[k], want[k], err[k], "affine_grad " + k)


def test_gradients_against_differences(ctx):
    """The loss sum(y * c) is linear in each argument by itself: the central difference along a direction is the gradient's
    product with it but for rounding -- 64-bit sums of a few thousand terms of size one, divided by a step of 1/2."""
    d = ref.make(11, (120, 33, 21, 6, 3, 5))
    d["slots"][1] = -1
    rng = np.random.default_rng(4)
    c = d["dy"]

    def loss(**kw):
        v = dict(d, **kw)
        return float((ctx.projection(v["x"], d["offsets"], v["w"], v["a"], v["b"], v["bias"], d["scale"], d["slots"]) * c).sum())

    g = ctx.projection_grad(d["x"], d["offsets"], d["w"], d["a"], d["b"], c, d["scale"], d["slots"])
    for k in g:
        v = rng.standard_normal(d[k].shape)
        diff = loss(**{k: d[k] + 0.25 * v}) - loss(**{k: d[k] - 0.25 * v})
        assert abs(diff / 0.5 - float((g[k] * v).sum())) <= 1e-9 * max(1.0, abs(diff)), k
    d["slots"][1] = 0

    def loss3(**kw):
        v = dict(d, **kw)
        return float((ctx.affine(v["x"], d["offsets"], v["w"], v["bias"], d["slots"]) * c).sum())

    d["w"], d["bias"] = d["w3"], d["bias2"]
    g = ctx.affine_grad(d["x"], d["offsets"], d["w"], c, d["slots"])
    for k in g:
        v = rng.standard_normal(d[k].shape)
        diff = loss3(**{k: d[k] + 0.25 * v}) - loss3(**{k: d[k] - 0.25 * v})
        assert abs(diff / 0.5 - float((g[k] * v).sum())) <= 1e-9 * max(1.0, abs(diff)), k


@pytest.mark.parametrize("kind", KINDS)
def test_rows_of_no_segment_stay(ctx, kind):
    """Rows before the first and behind the last segment keep what y and dx held (a NaN there included), and their x and dy are
    not part of any sum."""
    d = typed(ref.make(5, (90, 39, 24, 4, 4, 8), slots=False), kind)
    d["offsets"] = np.array([3, 20, 20, 57, 81], dtype=np.int64)
    for k in ("x", "dy", "y0", "dx0"):
        d[k][:3] = np.nan
        d[k][81:] = np.nan
    live = slice(3, 81)
    for y, want, err in (
            (ctx.affine(d["x"], d["offsets"], d["w3"], d["bias2"], out=d["y0"].copy()),
             *ref.affine(kind, d["x"], d["offsets"], d["w3"], d["bias2"], None, d["y0"])),
            (ctx.projection(d["x"], d["offsets"], d["w"], d["a"], d["b"], out=d["y0"].copy()),
             *ref.projection(kind, d["x"], d["offsets"], d["w"], d["a"], d["b"], None, None, None, d["y0"]))):
        assert np.isnan(y[:3]).all() and np.isnan(y[81:]).all()
        ref.check(y[live], want[live], err[live])
    fresh = ctx.affine(d["x"], d["offsets"], d["w3"], d["bias2"])
    assert not fresh[:3].any() and not fresh[81:].any()
    out = {"x": d["dx0"].copy(), "w": np.empty_like(d["w3"]), "bias": np.empty_like(d["bias2"])}
    got = ctx.affine_grad(d["x"], d["offsets"], d["w3"], d["dy"], out=out)
    want, err = ref.affine_grad(kind, d["x"], d["offsets"], d["w3"], d["dy"], None, d["dx0"])
    assert np.isnan(got["x"][:3]).all() and np.isnan(got["x"][81:]).all()
    ref.check(got["x"][live], want["x"][live], err["x"][live])
    for k in ("w", "bias"):
        ref.check(got[k], want[k], err[k], k)
    got = ctx.projection_grad(d["x"], d["offsets"], d["w"], d["a"], d["b"], d["dy"])
    want, err = ref.projection_grad(kind, d["x"], d["offsets"], d["w"], d["a"], d["b"], d["dy"], None, None, np.zeros_like(d["dx0"]))
    for k in got:
        ref.check(got[k], want[k], err[k], k)


@pytest.mark.parametrize("kind", KINDS)
def test_a_nan_stays_with_its_own(ctx, kind):
    """A diverged transform, adapter or row gives NaN where its products go, and nowhere else."""
    d = typed(ref.make(6, (100, 40, 24, 10, 5, 8)), kind)
    d["slots"] = np.array([0, 1, 2, 3, 4, 4, 3, 2, 1, 0], dtype=np.int32)
    d["offsets"] = np.arange(0, 101, 10).astype(np.int64)
    sick = np.zeros(100, dtype=bool)
    sick[10:20] = sick[80:90] = True                                     # rows of group 1
    for name in ("w3", "a", "b"):
        e = {k: v.copy() if isinstance(v, np.ndarray) else v for k, v in d.items()}
        e[name][1] = np.nan
        if name == "w3":
            y = ctx.affine(e["x"], e["offsets"], e["w3"], e["bias2"], e["slots"])
            dx = ctx.affine_grad(e["x"], e["offsets"], e["w3"], e["dy"], e["slots"], want=("x",))["x"]
            want = ref.affine(kind, d["x"], d["offsets"], d["w3"], d["bias2"], d["slots"], d["y0"])
            wantx, errx = (t["x"] for t in ref.affine_grad(kind, d["x"], d["offsets"], d["w3"], d["dy"], d["slots"], d["dx0"]))
        else:
            y = ctx.projection(e["x"], e["offsets"], e["w"], e["a"], e["b"], e["bias"], None, e["slots"])
            dx = ctx.projection_grad(e["x"], e["offsets"], e["w"], e["a"], e["b"], e["dy"], None, e["slots"], want=("x",))["x"]
            want = ref.projection(kind, d["x"], d["offsets"], d["w"], d["a"], d["b"], d["bias"], None, d["slots"], d["y0"])
            wantx, errx = (t["x"] for t in ref.projection_grad(kind, d["x"], d["offsets"], d["w"], d["a"], d["b"], d["dy"], None, d["slots"], d["dx0"]))
        assert np.isnan(y[sick]).all() and np.isnan(dx[sick]).all(), name
        ref.check(y[~sick], want[0][~sick], want[1][~sick], name)
        ref.check(dx[~sick], wantx[~sick], errx[~sick], name)
    e = dict(d, x=d["x"].copy())
    e["x"][33] = np.inf                                                  # a row of group 3
    y = ctx.affine(e["x"], e["offsets"], e["w3"], e["bias2"], e["slots"])
    assert not np.isfinite(y[33]).any()
    well = np.arange(100) != 33
    want = ref.affine(kind, d["x"], d["offsets"], d["w3"], d["bias2"], d["slots"], d["y0"])
    ref.check(y[well], want[0][well], want[1][well])
    g = ctx.affine_grad(e["x"], e["offsets"], e["w3"], e["dy"], e["slots"])["w"]
    assert not np.isfinite(g[3]).any() and np.isfinite(g[[0, 1, 2, 4]]).all()


def test_same_bits_every_time(ctx):
    d = typed(ref.make(7, (5000, 39, 39, 40, 6, 4)), "float32")
    a = ctx.affine_grad(d["x"], d["offsets"], d["w3"], d["dy"], d["slots"])
    for _ in range(3):
        b = ctx.affine_grad(d["x"], d["offsets"], d["w3"], d["dy"], d["slots"])
        for k in a:
            assert np.array_equal(a[k], b[k]), k


def test_nothing_to_do(ctx):
    """No rows, no segments, all segments empty: outputs of sums are zeros, y keeps its rows."""
    x, w, dy = np.zeros((0, 5)), np.ones((3, 4, 5)), np.zeros((0, 4))
    off = np.zeros(4, dtype=np.int64)
    assert ctx.affine(x, off, w).shape == (0, 4)
    g = ctx.affine_grad(x, off, w, dy, out={"x": np.zeros((0, 5)), "w": np.full((3, 4, 5), 7.0), "bias": np.full((3, 4), 7.0)})
    assert not g["w"].any() and not g["bias"].any()
    x, dy = np.ones((6, 5)), np.ones((6, 4))
    y = ctx.affine(x, off, w, out=np.full((6, 4), 3.0))                  # three empty segments
    assert (y == 3.0).all()
    none = np.zeros(1, dtype=np.int64)
    y = ctx.affine(x, none, w, slots=np.zeros(0, dtype=np.int32), out=np.full((6, 4), 3.0))
    assert (y == 3.0).all()
    a, b = np.ones((2, 3, 5)), np.ones((2, 4, 3))
    for off, slots in ((np.zeros(3, dtype=np.int64), None), (none, np.zeros(0, dtype=np.int32))):
        g = ctx.projection_grad(x, off, w[0], a, b, dy, slots=slots)
        assert not any(v.any() for v in g.values())
        assert (ctx.projection(x, off, w[0], a, b, slots=slots, out=np.full((6, 4), 3.0)) == 3.0).all()
    # no adapters at all: the projection alone
    y = ctx.projection(x, np.array([0, 6]), w[0], np.zeros((0, 3, 5)), np.zeros((0, 4, 3)), slots=np.array([-1], dtype=np.int32))
    assert (y == 5.0).all()
    g = ctx.projection_grad(x, np.array([0, 6]), w[0], np.zeros((0, 3, 5)), np.zeros((0, 4, 3)), dy, slots=np.array([-1], dtype=np.int32))
    assert (g["w"] == 6.0).all() and (g["x"] == 4.0).all() and g["a"].shape == (0, 3, 5)


def test_device_offsets_out_of_order_stay_in_bounds(ctx):
    """Offsets and slots in device memory are not looked at by the host: bad ones are brought into range by the kernels."""
    d = ref.make(8, (64, 16, 16, 6, 3, 4))
    up = ctx.to_device
    off = up(np.array([-50, 1 << 40, 10, 60, -(1 << 60), 1 << 62, 64], dtype=np.int64))
    sl = up(np.array([0, 99, -7, 1 << 30, 2, -(1 << 31)], dtype=np.int32))
    y = ctx.affine(up(d["x"]), off, up(d["w3"]), up(d["bias2"]), sl)
    g = ctx.affine_grad(up(d["x"]), off, up(d["w3"]), up(d["dy"]), sl)
    p = ctx.projection(up(d["x"]), off, up(d["w"]), up(d["a"]), up(d["b"]), slots=sl)
    h = ctx.projection_grad(up(d["x"]), off, up(d["w"]), up(d["a"]), up(d["b"]), up(d["dy"]), slots=sl)
    ctx.sync()
    assert y.shape == p.shape == (64, 16) and sorted(g) == ["bias", "w", "x"] and len(h) == 5
    # slots out of range, offsets in order: an affine row of such a segment stays, a projected one has no adapter
    off = np.array([0, 10, 20, 30, 40, 50, 64], dtype=np.int64)
    sl = np.array([0, 99, -7, 1, 2, -1], dtype=np.int32)
    y = ctx.affine(up(d["x"]), off, up(d["w3"]), slots=up(sl), out=up(d["y0"])).to_host()
    lost = np.r_[10:30, 50:64]
    assert np.array_equal(y[lost], d["y0"][lost])
    fixed = np.where((sl < 0) | (sl > 2), -1, sl)
    p = ctx.projection(up(d["x"]), off, up(d["w"]), up(d["a"]), up(d["b"]), slots=up(sl)).to_host()
    ref.check(p, *ref.projection("float64", d["x"], off, d["w"], d["a"], d["b"], None, None, fixed, d["y0"]))
    g = ctx.affine_grad(up(d["x"]), off, up(d["w3"]), up(d["dy"]), slots=up(sl))["w"].to_host()
    want = np.zeros_like(d["w3"])
    for s, k in enumerate(fixed):
        if k >= 0:
            want[k] += d["dy"][off[s]:off[s + 1]].T @ d["x"][off[s]:off[s + 1]]
    assert np.abs(g - want).max() <= 1e-12


def test_many_segments_and_groups(ctx):
    """More segments than one pass of the sort, more groups than one digit of it."""
    rng = np.random.default_rng(9)
    S, G, I, O = 5000, 700, 6, 5
    sizes = rng.integers(0, 4, S)
    off = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int64)
    sl = rng.integers(0, G, S).astype(np.int32)
    x, w, dy = rng.standard_normal((off[-1], I)), rng.standard_normal((G, O, I)), rng.standard_normal((off[-1], O))
    y = ctx.affine(x, off, w, slots=sl)
    ref.check(y, *ref.affine("float64", x, off, w, None, sl, np.zeros_like(y)))
    g = ctx.affine_grad(x, off, w, dy, sl)
    want, err = ref.affine_grad("float64", x, off, w, dy, sl, np.zeros_like(x))
    for k in want:
        ref.check(g[k], want[k], err[k], k)


def test_long_group_is_joined(ctx):
    """One group over many spans: 300,000 rows, each product 1 or -1, the sums exact."""
    F = 300000
    rng = np.random.default_rng(10)
    x, dy = rng.integers(0, 2, (F, 3)) * 2.0 - 1.0, rng.integers(0, 2, (F, 2)) * 2.0 - 1.0
    for kind in KINDS[:2]:
        g = ctx.affine_grad(x.astype(kind), np.array([0, F]), np.zeros((1, 2, 3), kind), dy.astype(kind), want=("w", "bias"))
        assert np.array_equal(g["w"][0], dy.T @ x) and np.array_equal(g["bias"][0], dy.sum(0))


def test_recognizer_with_speaker_transforms(tmp_path, synth, oracle):
    """MFCC -> speaker's transform -> decode, one utterance and a ragged batch, against the oracle's MFCC and decoding with the
    transform written out between them."""
    from lnasr.gmmhmm import GMMHMM
    from lnasr.recognizer import Recognizer
    from lnasr.transform import SpeakerTransforms
    rng = np.random.default_rng(13)
    pcm = [np.clip(synth.synth_signal(n, seed=30 + i) * 5, -32768, 32767).astype(np.int16) for i, n in enumerate((9000, 16000, 4400, 12345))]
    with np.errstate(divide="ignore"):
        feats = [oracle.mfcc(p.astype(np.float64))[2] for p in pcm]
    w = np.eye(39) + 0.1 * rng.standard_normal((3, 39, 39))
    bias = rng.standard_normal((3, 39))
    speakers = [2, 0, 1, 2]
    moved = [f @ w[k].T + bias[k] for f, k in zip(feats, speakers)]
    every = np.concatenate(moved)
    N, M, D = 8, 3, 39
    m = synth.synth_model(N, M, D, seed=5)
    pick = rng.choice(len(every), N * M, replace=False)
    mu, var = every[pick].reshape(N, M, D), np.broadcast_to(every.var(0) * 0.5 + 1.0, (N, M, D))
    si = np.zeros((N, M, D, D))
    si[:, :, np.arange(D), np.arange(D)] = var
    want = [oracle.decode_diag(f, m["A"], m["pi"], m["w"], mu, var) for f in moved]
    assert min(len(set(p.tolist())) for p in want) >= 3                    # the paths move between states
    GMMHMM(N, M, D, m["A"], m["pi"], m["w"], mu, si).save(str(tmp_path / "am.npz"))
    SpeakerTransforms(w, bias).save(str(tmp_path / "speakers.npz"))
    rec = Recognizer({"am": str(tmp_path / "am.npz"), "lm": None, "transform": str(tmp_path / "speakers.npz")})
    for p, k, path in zip(pcm, speakers, want):
        assert np.array_equal(rec.recognize(p, speaker=k), path)
    got = rec.recognize_batch(pcm, speakers)
    assert len(got) == 4 and all(np.array_equal(a, b) for a, b in zip(got, want))
    plain = Recognizer({"am": str(tmp_path / "am.npz")})
    assert plain.transforms is None
    assert all(np.array_equal(a, plain.recognize(p)) for a, p in zip(plain.recognize_batch(pcm), pcm))
    with pytest.raises(Exception, match="slots"):
        rec.recognize(pcm[0], speaker=3)


def test_calls_of_a_training_loop(ctx):
    """Forward, gradients and a step on the speakers' transforms under a quadratic loss, in fp64: along the gradient the loss differs
    by the gradient's square times the step, less the quadratic term, at every one of three steps."""
    d = ref.make(14, (400, 39, 39, 8, 3, 4))
    target = d["y0"]
    loss = lambda w, c: 0.5 * float(((ctx.affine(d["x"], d["offsets"], w, c, d["slots"]) - target) ** 2).sum())
    w, c = d["w3"].copy(), d["bias2"].copy()
    for _ in range(3):
        r = ctx.affine(d["x"], d["offsets"], w, c, d["slots"]) - target
        g = ctx.affine_grad(d["x"], d["offsets"], w, r, d["slots"], want=("w", "bias"))
        n = float((g["w"] ** 2).sum() + (g["bias"] ** 2).sum())
        curve = float((ctx.affine(d["x"], d["offsets"], g["w"], g["bias"], d["slots"]) ** 2).sum())
        h, before = 1e-4, loss(w, c)
        after = loss(w - h * g["w"], c - h * g["bias"])
        assert abs(before - after - (h * n - 0.5 * h * h * curve)) <= 1e-10 * before
        w, c = w - n / curve * g["w"], c - n / curve * g["bias"]


def test_refusals(ctx):
    from lnasr import _ffi
    x, w, off = np.zeros((6, 4)), np.zeros((2, 3, 4)), np.array([0, 2, 6])
    a, b, dy = np.zeros((2, 2, 4)), np.zeros((2, 3, 2)), np.zeros((6, 3))
    E = _ffi.LnasrError
    for err, match, call in (
            (E, "offsets fall", lambda: ctx.affine(x, [0, 4, 2], w)),
            (E, "offsets run", lambda: ctx.affine(x, [0, 4, 7], w)),
            (E, "offsets run", lambda: ctx.affine(x, [-1, 4, 6], w)),
            (E, r"slots\[1\] = 2", lambda: ctx.affine(x, off, w, slots=[0, 2])),
            (E, r"slots\[0\] = -1", lambda: ctx.affine(x, off, w, slots=[-1, 0])),
            (E, r"slots\[0\] = -2", lambda: ctx.projection(x, off, w[0], a, b, slots=[-2, 0])),
            (ValueError, "slots must have shape", lambda: ctx.affine(x, off, w, slots=[0])),
            (ValueError, "without slots", lambda: ctx.affine(x, [0, 6], w)),
            (ValueError, "x must have shape", lambda: ctx.affine(np.zeros((6, 5)), off, w)),
            (ValueError, "2 dimensions", lambda: ctx.affine(np.zeros(4), off, w)),
            (ValueError, "bias must have shape", lambda: ctx.affine(x, off, w, np.zeros((2, 4)))),
            (ValueError, "out must have shape", lambda: ctx.affine(x, off, w, out=np.zeros((6, 4)))),
            (E, "out is float32", lambda: ctx.affine(x, off, w, out=np.zeros((6, 3), np.float32))),
            (E, "writable", lambda: ctx.affine(x, off, w, out=np.zeros((6, 6))[:, :3])),
            (ValueError, "no gradient of 'y'", lambda: ctx.affine_grad(x, off, w, dy, want=("y",))),
            (E, "comes with that of w", lambda: ctx.affine_grad(x, off, w, dy, want=("bias",))),
            (ValueError, "dy must have shape", lambda: ctx.affine_grad(x, off, w, np.zeros((6, 4)))),
            (ValueError, "b must have shape", lambda: ctx.projection(x, off, w[0], a, np.zeros((2, 2, 3)))),
            (ValueError, "scale must have shape", lambda: ctx.projection(x, off, w[0], a, b, scale=np.zeros(3))),
            (E, "widths 0", lambda: ctx.affine(np.zeros((6, 0)), off, np.zeros((2, 3, 0)))),
            (E, "rank 0", lambda: ctx.projection(x, off, w[0], np.zeros((2, 0, 4)), np.zeros((2, 3, 0))))):
        with pytest.raises(err, match=match):
            call()
    d = ctx.to_device(x)
    sq = ctx.to_device(np.zeros((2, 4, 4)))
    with pytest.raises(E, match="shares memory"):
        ctx.affine(d, off, sq, out=d)
    with pytest.raises(E, match="shares memory"):
        ctx.affine_grad(d, off, sq, ctx.to_device(np.zeros((6, 4))), out={"x": d, "w": ctx.to_device(np.zeros((2, 4, 4)))})
    with pytest.raises(E, match="is float64"):
        ctx.affine(ctx.to_device(np.zeros((6, 4), np.float32)), off, ctx.to_device(w))
    with pytest.raises(E, match="is int32"):
        ctx.affine(ctx.to_device(np.zeros((6, 4), np.int32)), off, w)
    # the context works after all of that
    assert not ctx.affine(x, off, w).any()


def test_rows_of_empty_segments_with_slots(ctx):
    """No rows at all, but segments with groups: nothing to look up, every sum is zero."""
    w, a, b = np.ones((3, 4, 5)), np.ones((3, 2, 5)), np.ones((3, 4, 2))
    x, dy, off, sl = np.zeros((0, 5)), np.zeros((0, 4)), np.zeros(3, dtype=np.int64), np.array([2, 2], dtype=np.int32)
    assert ctx.affine(x, off, w, slots=sl).shape == ctx.projection(x, off, w[0], a, b, slots=sl).shape == (0, 4)
    for g in (ctx.affine_grad(x, off, w, dy, slots=sl), ctx.projection_grad(x, off, w[0], a, b, dy, slots=sl)):
        assert all(not v.any() for v in g.values())


def test_threads_share_a_context(ctx):
    """Two threads, one context: each call's launches share its workspaces and stay together."""
    import threading
    sizes = [(900, 72, 80, 4, 3, 16), (700, 80, 72, 5, 2, 40)]
    data = [ref.make(60 + i, size) for i, size in enumerate(sizes)]

    def run(d):
        y = ctx.projection(d["x"], d["offsets"], d["w"], d["a"], d["b"], d["bias"], d["scale"], d["slots"])
        g = ctx.projection_grad(d["x"], d["offsets"], d["w"], d["a"], d["b"], d["dy"], d["scale"], d["slots"])
        return [y] + [g[k] for k in sorted(g)]

    alone = [run(d) for d in data]
    wrong, failed = [], []

    def work(i):
        try:
            for _ in range(20):
                if not all(np.array_equal(u, v) for u, v in zip(run(data[i]), alone[i])):
                    wrong.append(i)
        except Exception as e:
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and not failed, (wrong, failed)


def test_arrays_of_another_context(ctx):
    """DeviceArrays of another context of the device: its work comes first, and it may read the result at once."""
    from lnasr import _ffi
    other = _ffi.Context(0)
    d = ref.make(62, (20000, 64, 48, 3, 3, 8), slots=False)
    x, w, y = other.to_device(d["x"]), other.to_device(d["w3"]), other.to_device(d["y0"])
    assert ctx.affine(x, d["offsets"], w, out=y) is y
    got = y.to_host()
    del x, w, y
    other.close()
    ref.check(got, *ref.affine("float64", d["x"], d["offsets"], d["w3"], None, None, d["y0"]))


def test_values_that_do_not_fit_are_refused(ctx):
    from lnasr import _ffi
    x, w, off = np.ones((6, 4)), [[[1.0] * 4] * 3] * 2, [0, 2, 6]
    assert (ctx.affine(x, off, w) == 4.0).all()                                     # lists become arrays
    for match, call in (("slots holds values", lambda: ctx.affine(x, off, w, slots=np.array([0, (1 << 32) + 1]))),
                        ("offsets holds values", lambda: ctx.affine(x, np.array([0, 1.5, 6]), w)),
                        ("offsets holds values", lambda: ctx.affine(x, np.array([0, 2, 1 << 63], dtype=np.uint64), w)),
                        ("array of complex", lambda: ctx.affine(x + 1j, off, w)),
                        ("array of str", lambda: ctx.affine(np.full((6, 4), "a"), off, w))):
        with pytest.raises(_ffi.LnasrError, match=match):
            call()


@pytest.mark.parametrize("size", [(9001, 840, 520, 6, 3, 24), (2000, 130, 200, 6, 3, 16), (90, 130, 200, 6, 3, 16)], ids=str)
def test_device_offsets_out_of_order_in_the_wide_forms(ctx, size):
    """The same at sizes that the tiles through LDS take: every offset is brought into range, whatever their order."""
    d = ref.make(63, size)
    F, S = size[0], size[3]
    bad = np.array([-50, 1 << 40, F // 3, F - 5, -(1 << 60), 1 << 62, F], dtype=np.int64)
    sl = np.array([0, 99, 1, 1 << 30, 2, 1], dtype=np.int32)
    up = lambda v, kind: ctx.to_device(np.ascontiguousarray(v, dtype=kind))
    for kind in ("float16", "float32"):
        x, dy, w3, w, a, b = (up(d[k], kind) for k in ("x", "dy", "w3", "w", "a", "b"))
        for off in (bad, bad[::-1].copy(), np.full(S + 1, F), np.array([7] * S + [F])):
            off, slots = ctx.to_device(off.astype(np.int64)), ctx.to_device(sl)
            y, p = ctx.affine(x, off, w3, slots=slots), ctx.projection(x, off, w, a, b, slots=slots)
            g, h = ctx.affine_grad(x, off, w3, dy, slots), ctx.projection_grad(x, off, w, a, b, dy, slots=slots)
            ctx.sync()
            assert y.shape == p.shape == (F, size[2]) and len(g) == 3 and len(h) == 5
    # the last of them, seven rows that belong to nobody, is in order
    want = d["y0"].astype("float32")
    got = ctx.affine(x, off, w3, slots=slots, out=up(want, "float32")).to_host()
    assert np.array_equal(got[:7], want[:7])


def everything(ctx, kind, d):
    y = ctx.projection(d["x"], d["offsets"], d["w"], d["a"], d["b"], d["bias"], d["scale"], d["slots"])
    ref.check(y, *ref.projection(kind, d["x"], d["offsets"], d["w"], d["a"], d["b"], d["bias"], d["scale"], d["slots"], d["y0"]), "projection")
    got = ctx.projection_grad(d["x"], d["offsets"], d["w"], d["a"], d["b"], d["dy"], d["scale"], d["slots"])
    want, err = ref.projection_grad(kind, d["x"], d["offsets"], d["w"], d["a"], d["b"], d["dy"], d["scale"], d["slots"], d["dx0"])
    for k in want:
        ref.check(got[k], want[k], err[k], "projection_grad " + k)
    if d["slots"] is not None:
        d["slots"] = np.maximum(d["slots"], 0)
    y = ctx.affine(d["x"], d["offsets"], d["w3"], d["bias2"], d["slots"])
    ref.check(y, *ref.affine(kind, d["x"], d["offsets"], d["w3"], d["bias2"], d["slots"], d["y0"]), "affine")
    got = ctx.affine_grad(d["x"], d["offsets"], d["w3"], d["dy"], d["slots"])
    want, err = ref.affine_grad(kind, d["x"], d["offsets"], d["w3"], d["dy"], d["slots"], d["dx0"])
    for k in want:
        ref.check(got[k], want[k], err[k], "affine_grad " + k)


@pytest.mark.parametrize("size,slots", [((20000, 1024, 1030, 90, 4, 9), True), ((20000, 1032, 1024, 70, 70, 8), False),
                                        ((16384, 72, 1030, 1, 1, 3), False), ((16640, 1024, 1024, 2, 1, 16), True)], ids=str)
def test_wide_tiles_of_many_segments_and_of_one(ctx, size, slots):
    """The largest tiles where the segments are more than a wave's lanes, and where there are one or two."""
    everything(ctx, "float16", typed(ref.make(70, size, slots=slots), "float16"))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", [(3, 1, 70001, 2, 2, 3), (3, 70001, 1, 2, 2, 3), (40, 24, 40, 5, 3, 300), (200, 351, 128, 6, 4, 12),
                                  (3000, 3, 700, 4, 3, 2), (3000, 700, 3, 4, 3, 2), (2500, 30, 30, 160, 9, 2), (2500, 30, 30, 900, 40, 2)], ids=str)
def test_extreme_widths_ranks_and_segments(ctx, kind, size):
    """One value in or out, ranks past both widths, narrow rows whose segments are as short as the pieces they are summed in."""
    everything(ctx, kind, typed(ref.make(71, size, negative=True), kind))


def test_inputs_and_outputs_of_different_places(ctx):
    """numpy in and DeviceArrays out, and the other way round."""
    d = ref.make(72, (300, 39, 40, 7, 3, 8))
    want, bound = ref.affine("float64", d["x"], d["offsets"], d["w3"], d["bias2"], d["slots"], d["y0"])
    out = ctx.to_device(d["y0"])
    assert ctx.affine(d["x"], d["offsets"], d["w3"], d["bias2"], d["slots"], out=out) is out
    ref.check(out.to_host(), want, bound)
    out = d["y0"].copy()
    assert ctx.affine(ctx.to_device(d["x"]), ctx.to_device(d["offsets"]), d["w3"], ctx.to_device(d["bias2"]), d["slots"], out=out) is out
    ref.check(out, want, bound)


@pytest.mark.parametrize("size,slots", [((16384, 128, 1024, 1, 1, 3), False), ((30000, 1024, 1030, 12, 5, 8), True)], ids=str)
def test_wide_tiles_of_few_segments_in_full_turns(ctx, size, slots):
    """The largest tiles where they fill the chip in whole turns (the sizes above leave a turn half empty)."""
    everything(ctx, "float16", typed(ref.make(73, size, slots=slots), "float16"))
