"""bfloat16 arrays without a library that knows them: 16-bit words in DeviceArrays, handed to the C entry points themselves."""
import ctypes as C

import numpy as np


def words(v):
    """float64 -> the nearest bfloat16 (ties to even), as uint16."""
    f = np.ascontiguousarray(v, dtype=np.float32)
    u = f.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    r[~np.isfinite(f)] = (f.view(np.uint32)[~np.isfinite(f)] >> 16).astype(np.uint16)
    return r


def values(w):
    return (w.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


class Calls:
    """The four operators on 16-bit inputs of one type ("float16" or "bfloat16"): float64 arrays of values in and out."""

    def __init__(self, ctx, kind):
        from lnasr import _ffi
        self.ctx, self.f, self.kind = ctx, _ffi, kind
        self.code = _ffi._CODES[kind]

    def round(self, v):
        """float64 values as the type holds them"""
        return v.astype(np.float16).astype(np.float64) if self.kind == "float16" else values(words(v))

    def up(self, v):
        if v is None:
            return None
        return self.ctx.to_device(v.astype(np.float16) if self.kind == "float16" else words(v))

    def down(self, d):
        h = d.to_host()
        return h.astype(np.float64) if self.kind == "float16" else values(h)

    @staticmethod
    def _p(d):
        return None if d is None else C.c_void_p(d.ptr)

    def projection(self, d):
        F, I = d["x"].shape
        O, G, R = d["w"].shape[0], d["a"].shape[0], d["a"].shape[1]
        h = [self.up(d[k]) for k in ("x", "w", "bias", "a", "b", "y0")]
        x, w, bias, a, b, y = h
        off, sl = self.ctx.to_device(d["offsets"]), None if d["slots"] is None else self.ctx.to_device(d["slots"])
        scale = self.ctx.to_device(d["scale"])
        self.f.check(self.f.lib().lnasr_projection(self.ctx.handle, self.code, x.ptr, F, I, I, off.ptr, sl and sl.ptr, len(d["offsets"]) - 1,
                                                   w.ptr, bias.ptr, O, a.ptr, b.ptr, scale.ptr, G, R, y.ptr, O))
        return self.down(y)

    def projection_grad(self, d):
        F, I = d["x"].shape
        O, G, R = d["w"].shape[0], d["a"].shape[0], d["a"].shape[1]
        x, w, a, b, dy, dx = (self.up(d[k]) for k in ("x", "w", "a", "b", "dy", "dx0"))
        off, sl = self.ctx.to_device(d["offsets"]), None if d["slots"] is None else self.ctx.to_device(d["slots"])
        scale = self.ctx.to_device(d["scale"])
        out = {"x": dx, "a": self.up(d["a"]), "b": self.up(d["b"]), "w": self.up(d["w"]), "bias": self.up(d["bias"])}
        self.f.check(self.f.lib().lnasr_projection_grad(
            self.ctx.handle, self.code, x.ptr, F, I, I, off.ptr, sl and sl.ptr, len(d["offsets"]) - 1, w.ptr, O, a.ptr, b.ptr, scale.ptr,
            G, R, dy.ptr, O, dx.ptr, I, out["a"].ptr, out["b"].ptr, out["w"].ptr, out["bias"].ptr))
        return {k: self.down(v) for k, v in out.items()}
