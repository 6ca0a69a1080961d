"""CPU: the feature transforms' entry points refuse before they touch a device; the plain forms of the GPU tests agree with
central differences and notice a planted mistake."""
import os
import re

import numpy as np
import pytest

import _transform_ref as ref
from conftest import REPO


def test_entry_points_refuse_a_null_context():
    from lnasr import _ffi
    l = _ffi.lib()
    z = 0
    assert l.lnasr_affine(None, 0, None, z, 1, z, None, None, z, None, None, z, 1, None, z) == -1
    assert l.lnasr_affine_grad(None, 0, None, z, 1, z, None, None, z, None, z, 1, None, z, None, z, None, None) == -1
    assert l.lnasr_projection(None, 0, None, z, 1, z, None, None, z, None, None, 1, None, None, None, z, 1, None, z) == -1
    assert l.lnasr_projection_grad(None, 0, None, z, 1, z, None, None, z, None, 1, None, None, None, z, 1, None, z, None, z, None,
                                   None, None, None) == -1
    assert b"null ctx" in l.lnasr_last_error()
    assert l.lnasr_ctx_use_stream(None, None, 1) == -1


def test_table_matches_the_header():
    from lnasr import _ffi
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(REPO, "include", "lnasr_transform.h")).read(), flags=re.S)
    assert sorted(_ffi.TRANSFORM_SIGNATURES) == sorted(set(re.findall(r"\b(lnasr_[a-z0-9_]+)\s*\(", text)))
    assert not set(_ffi.TRANSFORM_SIGNATURES) & set(_ffi.SIGNATURES)
    for name, args in _ffi.TRANSFORM_SIGNATURES.items():                            # one type for each declared argument
        declared = re.search(r"\b%s\s*\(([^)]*)\)" % name, text).group(1)
        assert len(args) == declared.count(",") + 1, name
        assert hasattr(_ffi.lib(), name)


class _Ctx:
    device = 0
    _tensors_checked = True


def test_arguments_are_checked_before_the_library_is_called():
    from lnasr import _ffi
    arg = lambda x, nd, **kw: _ffi._Arg(_Ctx, x, "x", nd, **kw)
    assert arg([[1, 2], [3, 4]], 2).kind == "float64"
    assert arg(np.zeros((2, 3), np.float16), 2).ld == 3
    assert arg(np.zeros((4, 6), np.float32)[:, :3], 2).ld == 3                     # copied
    with pytest.raises(ValueError, match="dimensions"):
        arg(np.zeros(3), 2)
    with pytest.raises(_ffi.LnasrError, match="writable"):
        arg([1.0], 1, out=True)
    ro = np.zeros((2, 2))
    ro.flags.writeable = False
    with pytest.raises(_ffi.LnasrError, match="writable"):
        arg(ro, 2, out=True)
    with pytest.raises(_ffi.LnasrError, match="expected float64"):
        arg(np.zeros((2, 2), np.float32), 2, like=arg(np.zeros((2, 2)), 2), out=True)

    class Tensor:
        """what the binding asks of a tensor of another library"""
        is_cuda, dtype, shape = True, "torch.bfloat16", (4, 3)
        strides, dev = (8, 1), 0
        data_ptr = lambda self: 4096
        get_device = lambda self: self.dev
        stride = lambda self: self.strides
        is_contiguous = lambda self: self.strides == (3, 1)

    t = Tensor()
    assert (arg(t, 2).kind, arg(t, 2).ld) == ("bfloat16", 8)
    t.strides = (1, 4)
    with pytest.raises(_ffi.LnasrError, match="contiguous"):
        arg(t, 2)
    t.strides = (0, 1)                                                              # one row seen four times
    with pytest.raises(_ffi.LnasrError, match="contiguous"):
        arg(t, 2)
    t.strides, t.dev = (3, 1), 1
    with pytest.raises(_ffi.LnasrError, match="device 1"):
        arg(t, 2)
    t.dev, t.dtype = 0, "torch.int64"
    with pytest.raises(_ffi.LnasrError, match="int64"):
        arg(t, 2)


def test_plain_forms_against_differences():
    d = ref.make(1, (40, 9, 7, 5, 3, 2), negative=True)
    rng = np.random.default_rng(2)
    y = lambda v: ref.projection("float64", v["x"], d["offsets"], v["w"], v["a"], v["b"], v["bias"], d["scale"], d["slots"], d["y0"])[0]
    g, err = ref.projection_grad("float64", d["x"], d["offsets"], d["w"], d["a"], d["b"], d["dy"], d["scale"], d["slots"], d["dx0"])
    for k in g:
        v = rng.standard_normal(d[k].shape)
        diff = ((y(dict(d, **{k: d[k] + v})) - y(dict(d, **{k: d[k] - v}))) * d["dy"]).sum() / 2
        assert abs(diff - (g[k] * v).sum()) <= 1e-10 * max(1.0, abs(diff)), k
    ref.check(g["a"], g["a"], err["a"])
    wrong = g["a"].copy()
    wrong.flat[3] += 1e-9                                                           # a planted mistake
    with pytest.raises(AssertionError, match="1 of"):
        ref.check(wrong, g["a"], err["a"])
