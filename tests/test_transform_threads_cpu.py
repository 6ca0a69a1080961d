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
