"""What the 8-bit KV cache's entries and wrapper refuse before any device call: addresses that a kernel could not read."""
import ctypes as C

import pytest
import torch

from opennpu_b200 import kv8
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


@pytest.mark.parametrize("fn", ["append", "read", "attn"])
def test_rows_whose_counts_pass_32_bits_are_refused(fn, monkeypatch):
    """The kernels step up to 2100 rows past a sequence's last in 32 bits."""
    rows = (1 << 31) - 4095
    monkeypatch.setattr(DESC, "rows", rows)
    for name, stride in (("hs", rows * 64), ("bs", 4 * rows * 64), ("shs", 1 << 26), ("sbs", 1 << 28)):
        monkeypatch.setattr(DESC, name, stride)
    assert call(fn) < 0 and "2^31 - 4096" in L.last_error()


class FakeCuda:
    """What the wrapper looks at of a dense CUDA tensor on device 1."""
    is_cuda, device = True, torch.device("cuda", 1)

    def __init__(self, dtype, *shape):
        self.dtype, self.shape = dtype, torch.Size(shape)

    def dim(self):
        return len(self.shape)

    def stride(self, i=None):
        s = torch.empty(self.shape, device="meta").stride()
        return s if i is None else s[i]

    def get_device(self):
        return 1

    def data_ptr(self):
        return 1 << 20


def test_a_cache_on_another_device_than_the_current_one_is_refused(monkeypatch):
    """The kernels run on the library's device, which the current one has to be, and would read the cache's addresses there."""
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(L, "require_device", lambda: pytest.fail("the cache was taken"))
    k, s = FakeCuda(torch.int8, 2, 4, 100, 64), FakeCuda(torch.float32, 2, 4, 4)
    with pytest.raises(L.OnpuError, match="current device"):
        kv8.KVCache8.from_tensors(k, k, s, s)


@pytest.mark.parametrize("block", [0, 8, -32, 48, None])
def test_a_bad_block_is_refused_before_anything_is_allocated(block):
    with pytest.raises(L.OnpuError, match="block"):
        kv8.KVCache8(1, 1, 32, 64, block=block)
