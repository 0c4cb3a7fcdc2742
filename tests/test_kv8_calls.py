"""What the 8-bit KV cache's entries refuse before any device call: pointers that a kernel could not read."""
import ctypes as C

import pytest

from opennpu_b200 import libonpu as L

DESC = L.Kv8Cache(1 << 20, 1 << 21, 1 << 22, 1 << 23, 2, 4, 100, 64, 4 * 100 * 64, 100 * 64, 64, 16, 4, 32)
ROWS, OUT, POS, WS, ODD = 1 << 24, 1 << 25, 1 << 26, 1 << 27, (1 << 28) + 2


def call(fn, pos=POS, cnt=None, mask=None, sinks=None):
    lib, r = L.load(), C.addressof(DESC)
    if fn == "append":
        return lib.onpu_kv8_append_dev(r, ROWS, 256, OUT, 256, 3, 1, pos, cnt, None)
    if fn == "read":
        return lib.onpu_kv8_read_dev(r, ROWS, 256, OUT, 256, 3, 1, pos, cnt, None)
    return lib.onpu_kv8_attn_dev(r, ROWS, 512, 8, 3, 1, pos, cnt, mask, 0, 0, sinks, 0.125, OUT, 512, WS, None)


@pytest.mark.parametrize("fn,bad", [("append", "pos"), ("append", "cnt"), ("read", "pos"), ("read", "cnt"), ("attn", "pos"),
                                    ("attn", "cnt"), ("attn", "mask"), ("attn", "sinks")])
def test_words_that_are_not_4_byte_aligned_are_refused(fn, bad):
    assert call(fn, **{bad: ODD}) < 0
    assert f"onpu_kv8_{fn}_dev" in L.last_error() and "4-byte aligned" in L.last_error()
