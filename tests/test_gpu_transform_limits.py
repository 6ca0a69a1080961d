"""GPU: feature transforms where a size or a stride passes what one launch, one offset or one wave's LDS holds."""
import ctypes as C

import numpy as np
import pytest

import _transform_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from lnasr import _ffi
    c = _ffi.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("kind", ["float64", "float32", "float16"])
def test_matrix_gradients_of_rows_far_apart(ctx, kind):
    """Rows 2^24 values apart, long segments, groups that do not lie in their order: each group sums its own rows."""
    from lnasr import _ffi
    e = np.dtype(kind).itemsize
    per, far, I, O, R = 512 // e + 3, 1 << 24, 24, 20, 5
    rows = 2 * per
    d = ref.make(1, (rows, I, O, 2, 3, R))
    d["offsets"], d["slots"] = np.array([0, per, rows], dtype=np.int64), np.array([2, 0], dtype=np.int32)
    d = {k: v if k in ("offsets", "slots", "scale") else v.astype(kind) for k, v in d.items()}
    l = _ffi.lib()
    room = _ffi.DeviceArray(ctx, ((rows - 1) * far + I,), kind)
    for r in range(rows):                                                # (the rest is never looked at)
        _ffi.check(l.lnasr_memcpy_h2d(ctx.handle, C.c_void_p(room.ptr + r * far * e), np.ascontiguousarray(d["x"][r]).ctypes.data, I * e))
    w3, w, a, b, dy, off, sl, scale = (ctx.to_device(d[k]) for k in ("w3", "w", "a", "b", "dy", "offsets", "slots", "scale"))
    dw, db = ctx.to_device(np.full_like(d["w3"], np.nan)), ctx.to_device(np.full_like(d["bias2"], np.nan))
    code = _ffi._CODES[kind]
    _ffi.check(l.lnasr_affine_grad(ctx.handle, code, room.ptr, rows, I, far, off.ptr, sl.ptr, 2, w3.ptr, 3, O, dy.ptr, O, None, 0, dw.ptr, db.ptr))
    want, err = ref.affine_grad(kind, d["x"], d["offsets"], d["w3"], d["dy"], d["slots"], d["dx0"])
    ref.check(dw.to_host(), want["w"], err["w"], "w")
    ref.check(db.to_host(), want["bias"], err["bias"], "bias")
    da, db = ctx.to_device(np.full_like(d["a"], np.nan)), ctx.to_device(np.full_like(d["b"], np.nan))
    dws = ctx.to_device(np.full_like(d["w"], np.nan))
    _ffi.check(l.lnasr_projection_grad(ctx.handle, code, room.ptr, rows, I, far, off.ptr, sl.ptr, 2, w.ptr, O, a.ptr, b.ptr, scale.ptr, 3, R,
                                       dy.ptr, O, None, 0, da.ptr, db.ptr, dws.ptr, None))
    want, err = ref.projection_grad(kind, d["x"], d["offsets"], d["w"], d["a"], d["b"], d["dy"], d["scale"], d["slots"], d["dx0"])
    for k, v in (("a", da), ("b", db), ("w", dws)):
        ref.check(v.to_host(), want[k], err[k], k)
    room.free()


def check_columns(kind, x, got, w, slots, what):
    """got[r] = w[slots[r]] x[r] for one-row segments, as _transform_ref has it, some rows at a time"""
    for at in range(0, len(x), 8192):
        r = slice(at, min(at + 8192, len(x)))
        n = r.stop - at
        ref.check(got[r], *ref.affine(kind, x[r], np.arange(n + 1), w, None, slots[r], np.zeros((n, w.shape[1]))), what)


@pytest.mark.parametrize("kind", ["float32", "float16"])
def test_more_work_items_than_one_launch_takes(ctx, kind):
    """66,000 one-row segments of 2048 results: 9 million blocks of 512 threads, past 2^32 items."""
    rng = np.random.default_rng(2)
    F, K, N, G = 66000, 12, 2048, 3
    sl = rng.integers(0, G, F).astype(np.int32)
    off = np.arange(F + 1, dtype=np.int64)
    x, w = rng.standard_normal((F, K)).astype(kind), rng.standard_normal((G, N, K)).astype(kind)
    y = ctx.affine(ctx.to_device(x), off, ctx.to_device(w), slots=sl).to_host()
    check_columns(kind, x, y, w, sl, "y")
    wt = np.ascontiguousarray(w.transpose(0, 2, 1))                       # [G, K, N]: dx = wt^T dy has the same values
    g = ctx.affine_grad(ctx.to_device(np.ones((F, N), kind)), off, ctx.to_device(wt), ctx.to_device(x), sl, want=("x",))["x"].to_host()
    check_columns(kind, x, g, w, sl, "dx")


def test_more_groups_than_one_launch_has_blocks(ctx):
    """17 million groups of one value: past 2^32 items in the gradients and in the join of their sums."""
    G = 17_000_000
    x = (np.arange(G) % 7 - 3).astype(np.float32).reshape(G, 1)
    dy = (np.arange(G) % 5 - 2).astype(np.float32).reshape(G, 1)
    off = np.arange(G + 1, dtype=np.int64)
    off[1:1999] = 1999                                                    # a long group, and some of none
    want = (x * dy).astype(np.float64).ravel()
    want[0] = want[:1999].sum()
    want[1:1999] = 0
    g = ctx.affine_grad(x, off, np.zeros((G, 1, 1), np.float32), dy, want=("w",))["w"].ravel()
    assert np.array_equal(g, want)


@pytest.mark.parametrize("kind", ["float64", "float32", "float16"])
@pytest.mark.parametrize("K", [1, 9, 15, 16, 17, 33, 40, 41, 48, 49, 63, 64])
def test_narrow_rows_of_every_fragment_width(ctx, kind, K):
    """Rows whose fragments are read past the row's end, few results and many: all of it in the wave's own LDS (the build checks that
    for every width), and none of it in a result."""
    for N in (1, 16, 17, 64):
        d = ref.make(3, (333, K, N, 5, 3, 2))
        d = {k: v if k in ("offsets", "slots", "scale") else v.astype(kind) for k, v in d.items()}
        y = ctx.affine(d["x"], d["offsets"], d["w3"], d["bias2"], d["slots"], out=d["y0"].copy())
        ref.check(y, *ref.affine(kind, d["x"], d["offsets"], d["w3"], d["bias2"], d["slots"], d["y0"]), "y")
        y = ctx.affine(d["x"], d["offsets"], d["w3"], None, d["slots"], out=d["y0"].copy())
        ref.check(y, *ref.affine(kind, d["x"], d["offsets"], d["w3"], None, d["slots"], d["y0"]), "y without bias")


def test_no_segments_and_a_null_pointer_for_their_slots(ctx):
    """An empty tensor of slots has no memory: a batch without segments is one all the same."""
    from lnasr import _ffi
    l = _ffi.lib()
    x, dy, w, a, b = (ctx.to_device(np.ones(s)) for s in ((6, 5), (6, 4), (3, 4, 5), (3, 2, 5), (3, 4, 2)))
    off, y = ctx.to_device(np.zeros(1, dtype=np.int64)), ctx.to_device(np.full((6, 4), 7.0))
    dw, db = ctx.to_device(np.full((3, 4, 5), np.nan)), ctx.to_device(np.full((3, 4), np.nan))
    _ffi.check(l.lnasr_affine(ctx.handle, 0, x.ptr, 6, 5, 5, off.ptr, None, 0, w.ptr, None, 3, 4, y.ptr, 4))
    _ffi.check(l.lnasr_affine_grad(ctx.handle, 0, x.ptr, 6, 5, 5, off.ptr, None, 0, w.ptr, 3, 4, dy.ptr, 4, None, 0, dw.ptr, db.ptr))
    assert (y.to_host() == 7.0).all() and not dw.to_host().any() and not db.to_host().any()
    da, d2 = ctx.to_device(np.full((3, 2, 5), np.nan)), ctx.to_device(np.full((3, 4, 2), np.nan))
    _ffi.check(l.lnasr_projection(ctx.handle, 0, x.ptr, 6, 5, 5, off.ptr, None, 0, w.ptr, None, 4, a.ptr, b.ptr, None, 3, 2, y.ptr, 4))
    _ffi.check(l.lnasr_projection_grad(ctx.handle, 0, x.ptr, 6, 5, 5, off.ptr, None, 0, w.ptr, 4, a.ptr, b.ptr, None, 3, 2, dy.ptr, 4,
                                       None, 0, da.ptr, d2.ptr, None, None))
    assert (y.to_host() == 7.0).all() and not da.to_host().any() and not d2.to_host().any()
