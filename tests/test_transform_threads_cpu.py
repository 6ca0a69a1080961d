"""CPU: what threads that share a context for the feature transforms are promised."""
import os
import re

from conftest import REPO

CSRC = os.path.join(REPO, "ln-asr_amd", "csrc")


def body(text, name):
    """The source of function `name` from its definition to the closing brace in the first column."""
    at = re.search(r"^int %s\([^;{]*\{" % name, text, re.M)
    return text[at.end():text.index("\n}", at.end())]


def test_entry_points_change_the_context_only_under_its_lock():
    from lnasr import _ffi
    text = open(os.path.join(CSRC, "transform.hip")).read() + open(os.path.join(CSRC, "ctx.hip")).read()
    changes = re.compile(r"(\+\+|--)\(?ctx\)?->|\bctx->\w+(\.\w+)?\s*([+-]?=)[^=]|LN_ENTER|LN_LAUNCH|transform_ws|c\.begin")
    for name in _ffi.TRANSFORM_SIGNATURES:
        b = body(text, name)
        lock = re.search(r"Call c\(ctx\);|lock_guard<std::mutex> lock\(ctx->tr_mutex\);", b)
        assert lock, name
        assert not changes.search(b[:lock.start()]), name
    macro = re.search(r"#define LN_ENTER\(ctx\)(.*?)while \(0\)", open(os.path.join(CSRC, "common.h")).read(), re.S).group(1)
    assert "++(ctx)->" in macro                                    # LN_ENTER counts the call, without a lock


class _Lib:
    """The library as far as the choice of streams goes: what is enqueued where, and what waits."""

    def __init__(self):
        self.said, self.capturing = [], 0

    def lnasr_ctx_use_stream(self, handle, stream, own):
        self.said.append(("stream", None if own else stream))
        return 0

    def lnasr_ctx_capturing(self, handle):
        return self.capturing

    def __getattr__(self, name):
        return lambda *args: self.said.append(name) or 0


class _Tensor:
    is_cuda, dtype, shape = True, "torch.float32", (4, 3)
    data_ptr = lambda self: 4096
    get_device = lambda self: 0
    stride = lambda self: (3, 1)
    is_contiguous = lambda self: True


def in_thread(f):
    import threading
    failed = []

    def run():
        try:
            f()
        except BaseException as e:
            failed.append(e)
    t = threading.Thread(target=run)
    t.start()
    t.join()
    if failed:
        raise failed[0]


def test_a_threads_calls_go_to_the_stream_it_chose(monkeypatch):
    """Two threads, two streams, one context: each call is enqueued on its own thread's stream; a thread that chose none waits."""
    from lnasr import _ffi
    l = _Lib()
    monkeypatch.setattr(_ffi, "lib", lambda: l)
    monkeypatch.setattr(_ffi.Context, "__del__", lambda self: None, raising=False)
    ctx = _ffi.Context(0)
    ctx._tensors_checked = True
    x = lambda: _ffi._Arg(ctx, _Tensor(), "x", 2)

    def call():
        l.said.clear()
        ctx._call(l.lnasr_affine, (x(),))
        return list(l.said)

    wait = ["lnasr_device_sync", "lnasr_affine", "lnasr_sync"]
    assert call() == wait                                          # nobody has chosen
    ctx.use_stream(11)
    assert call() == ["lnasr_affine"]

    def other():
        assert call() == wait                                      # a thread that chose none
        ctx.use_stream(22)
        assert call() == ["lnasr_affine"]

    in_thread(other)
    assert call() == [("stream", 11), "lnasr_affine"]              # back to this thread's
    assert call() == ["lnasr_affine"]
    l.capturing = 1
    in_thread(lambda: (call() == ["lnasr_affine"]) or (_ for _ in ()).throw(AssertionError(l.said)))   # cannot wait
    l.capturing = 0
    ctx.use_stream(None)
    assert call() == wait
    in_thread(lambda: ctx.use_stream(22))
    assert call() == wait
