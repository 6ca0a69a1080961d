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
