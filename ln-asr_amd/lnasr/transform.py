"""Feature transforms between the front end and the models: affine maps per speaker or class, and a projection that all rows
share with a low-rank adapter per speaker beside it, with the gradients that train them (csrc/transform*.hip).  The reference
has none; `Recognizer` applies an affine bank between MFCC and decoding.

Rows are packed, as `MFCC.calc_mfcc_batch` returns features: segment s (an utterance, a request) holds rows
offsets[s] .. offsets[s+1]-1.  `slots` names the group (speaker) of each segment; without it segment s is group s.  Rows outside
offsets[0] .. offsets[-1] are left as they were in `out`, and are zeros in an array made here.

Arrays are numpy arrays, `DeviceArray`s, or GPU tensors of another library (torch's, which is not imported here: a tensor only
has to have data_ptr(), shape, dtype, stride()); what comes back is of the same kind as x.  x, matrices and results share one
type: float64, float32, float16 or (tensors) bfloat16.  Sums are held in 64 bits for float64 and in 32 for the others.  Rows may
be strided (a slice of columns); matrices are contiguous.  numpy arrays are converted to the type of x.  Results may be written
into `out`, which must not overlap an input (nor lie beside it in the columns of one buffer).  With GPU tensors, choose their
stream first (`ctx.use_stream`, in each thread that calls) and import their library before lnasr; in a thread that chose none, and
for `DeviceArray`s of another context, a call waits for the device before it begins and until it is done.  Calls are not recorded
by torch's autograd: a tensor that requires a gradient is refused unless recording is off, as under `torch.no_grad()` and in the
forward and backward of a `torch.autograd.Function`, where these functions and their gradients belong.
"""
import numpy as np

from ._ffi import default_ctx
from .hmm import _load, _save


def affine(x, offsets, w, bias=None, slots=None, out=None, *, ctx=None):
    """y[r] = w[k] x[r] + bias[k], k the group of row r.  x [F, din], w [G, dout, din], bias [G, dout] -> [F, dout]."""
    return (ctx or default_ctx()).affine(x, offsets, w, bias, slots, out)


def affine_grad(x, offsets, w, dy, slots=None, want=("x", "w", "bias"), out=None, *, ctx=None):
    """From dy [F, dout], the gradient of a loss by y: a dict of the gradients by "x" [F, din], "w" [G, dout, din] and "bias"
    [G, dout] (zeros for a group without rows).  want: which of them; or out: a dict of arrays to write exactly those into.
    "bias" comes with "w" only."""
    return (ctx or default_ctx()).affine_grad(x, offsets, w, dy, slots, want, out)


def projection(x, offsets, w, a, b, bias=None, scale=None, slots=None, out=None, *, ctx=None):
    """y[r] = w x[r] + bias + scale[k] b[k] (a[k] x[r]).  w [dout, din], bias [dout], a [G, rank, din], b [G, dout, rank], scale
    [G] float64 (default 1); slot -1: no adapter.  The middle, scale a x, is held in 64 bits for float64 and in 32 for the others."""
    return (ctx or default_ctx()).projection(x, offsets, w, a, b, bias, scale, slots, out)


def projection_grad(x, offsets, w, a, b, dy, scale=None, slots=None, want=("x", "a", "b", "w", "bias"), out=None, *, ctx=None):
    """The gradients of `projection` by "x", "a", "b", "w" and "bias", as `affine_grad` returns them; leave "w" and "bias" out to
    train adapters beside a frozen projection."""
    return (ctx or default_ctx()).projection_grad(x, offsets, w, a, b, dy, scale, slots, want, out)


class SpeakerTransforms:
    """A bank of affine feature transforms, one per speaker: `w` [G, dout, din] and `bias` [G, dout] in float64, kept on the device.
    `Recognizer` applies one between MFCC and decoding."""

    def __init__(self, w=None, bias=None, *, ctx=None):
        self._ctx = ctx
        self._set(w, bias)

    def _set(self, w, bias):
        self._held = None
        if w is None:
            self.w = self.bias = None
            return
        self.w = np.ascontiguousarray(w, dtype=np.float64)
        if self.w.ndim != 3:
            raise ValueError("w must have shape (speakers, dout, din), got %s" % (self.w.shape,))
        self.bias = np.zeros(self.w.shape[:2]) if bias is None else np.ascontiguousarray(bias, dtype=np.float64)
        if self.bias.shape != self.w.shape[:2]:
            raise ValueError("bias must have shape %s, got %s" % (self.w.shape[:2], self.bias.shape))

    @property
    def ctx(self):
        if self._ctx is None:
            self._ctx = default_ctx()
        return self._ctx

    def apply(self, features, offsets, speakers=None, out=None):
        """Features [F, din] of utterances (rows offsets[u] .. offsets[u+1]-1, float64: a numpy array or a DeviceArray) -> [F, dout].
        speakers [U]: the speaker of each; without it utterance u is speaker u's.  To change w or bias, make a new bank or `load`."""
        if self.w is None:
            raise ValueError("no transforms: give w, or load them")
        if self._held is None:
            self._held = (self.ctx.to_device(self.w), self.ctx.to_device(self.bias))
        return self.ctx.affine(features, offsets, *self._held, slots=speakers, out=out)

    def save(self, filename):
        """Datasets 'w' and 'bias', in the files the models use."""
        _save(filename, {"w": self.w, "bias": self.bias})

    def load(self, filename):
        d = _load(filename, ("w", "bias"))
        self._set(d["w"], d["bias"])
