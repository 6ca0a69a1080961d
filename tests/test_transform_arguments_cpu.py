"""CPU: arguments of the feature transforms that are refused, or taken for what they are, before the library is called."""
import sys
import types

import numpy as np
import pytest


class _Ctx:
    device = 0
    _tensors_checked = True


class _Tensor:
    is_cuda, dtype, shape, requires_grad = True, "torch.float32", (4, 3), True
    data_ptr = lambda self: 4096
    get_device = lambda self: 0
    stride = lambda self: (3, 1)
    is_contiguous = lambda self: True


def test_a_tensor_that_requires_a_gradient_is_refused_where_that_is_recorded(monkeypatch):
    from lnasr import _ffi
    arg = lambda: _ffi._Arg(_Ctx, _Tensor(), "w", 2)
    on = types.SimpleNamespace(is_grad_enabled=lambda: True)
    monkeypatch.setitem(sys.modules, "torch", on)
    with pytest.raises(_ffi.LnasrError, match="w requires a gradient"):
        arg()
    on.is_grad_enabled = lambda: False                             # no_grad(), or inside a Function
    assert arg().kind == "float32"
    monkeypatch.setattr(_Tensor, "requires_grad", False)
    on.is_grad_enabled = lambda: True
    assert arg().kind == "float32"


def test_an_output_of_another_byte_order_is_refused():
    """Its type has the same name, but results written there would be other numbers; an input is converted."""
    from lnasr import _ffi
    other = np.dtype(np.float64).newbyteorder()
    assert other.name == "float64"
    with pytest.raises(_ffi.LnasrError, match="writable"):
        _ffi._Arg(_Ctx, np.zeros((2, 3), other), "out", 2, out=True)
    a = _ffi._Arg(_Ctx, np.ones((2, 3), other), "x", 2)
    assert a.obj.dtype.isnative and a.obj.sum() == 6


class _Bank:
    """Stands for SpeakerTransforms: checks the speakers as the binding does."""

    def apply(self, features, offsets, speakers=None, out=None):
        from lnasr import _ffi
        self.seen = _ffi._Arg(_Ctx, speakers, "slots", 1, like="int32").obj.tolist()
        raise StopIteration


class _Front:
    """Stands for the front end and the model as far as `Recognizer` goes before it applies the transforms."""
    _cfg = lambda self: (None, None, None)
    to_device = lambda self, x: x
    mfcc = lambda self, *a: (None, None, np.zeros((4, 2)), np.array([0, 2, 4]))
    ctx = property(lambda self: self)


def test_speakers_are_whole_numbers():
    """1.7 is no speaker: it is refused, not cut down to speaker 1."""
    from lnasr import _ffi
    from lnasr.recognizer import Recognizer
    r = Recognizer.__new__(Recognizer)
    r.am, r.transforms = types.SimpleNamespace(mfcc=_Front(), gmmhmm=_Front()), _Bank()
    pcm = np.zeros(400, np.int16)
    for call in (lambda k: r.recognize(pcm, k), lambda k: r.recognize_batch([pcm, pcm], [0, k])):
        with pytest.raises(StopIteration):
            call(1)
        assert r.transforms.seen[-1] == 1
        for bad in (1.7, (1 << 32) + 1):
            with pytest.raises(_ffi.LnasrError, match="not int32"):
                call(bad)
