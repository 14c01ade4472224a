"""tpfm_prepare takes the old weights away before the new ones are there. If a
step between fails (no memory), a forward must be refused, not run on null
weights: the handle stops being ready before the first buffer goes, and is
ready again after the last step. The failure cannot be made on the host, so
the order is read in the source."""
import os
import re

from conftest import PKG


def body(text, start):
    """the function that begins with `start`, to its closing brace in column 0"""
    at = text.index(start)
    return text[at:text.index("\n}\n", at)]


def test_not_ready_before_the_first_buffer_goes():
    with open(os.path.join(PKG, "csrc", "tpfm_api.cu")) as f:
        f = body(f.read(), "int tpfm_prepare(tpfm_ctx *c) {")
    off, on = f.index("c->wready = false;"), f.index("c->wready = true;")
    assert f.count("wready") == 2
    assert off < min(m.start() for m in re.finditer(r"cudaFree|cudaGraphExecDestroy", f))
    assert on > max(m.start() for m in re.finditer(r"return -1", f))
