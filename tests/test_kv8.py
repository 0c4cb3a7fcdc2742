"""The 8-bit KV cache without a GPU: what the C entries and the wrapper refuse, and the oracle's own
definition (oracle.kv8_*) on cases worked out by hand."""
import ctypes as C

import numpy as np
import pytest
import torch

from opennpu_b200 import kv8
from opennpu_b200 import libonpu as L
from oracle import oracle as O

GOOD = dict(k=1 << 20, v=1 << 21, k_scale=1 << 22, v_scale=1 << 23, batch=2, heads=4, rows=100, dim=64, bs=4 * 100 * 64,
            hs=100 * 64, rs=64, sbs=16, shs=4, block=32)


def desc(**kw):
    return L.Kv8Cache(**{**GOOD, **kw})


def call(fn, d, rows=1 << 24, ld=256, T=3, bf16=1, pos=1 << 25, Hq=8, ws=1 << 26, out=1 << 24):
    lib, r = L.load(), None if d is None else C.addressof(d)
    if fn == "append":
        return lib.onpu_kv8_append_dev(r, rows, ld, rows, ld, T, bf16, pos, None, None)
    if fn == "read":
        return lib.onpu_kv8_read_dev(r, rows, ld, rows, ld, T, bf16, pos, None, None)
    return lib.onpu_kv8_attn_dev(r, rows, 2 * ld, Hq, T, bf16, pos, None, None, 0, 0, None, 0.125, out, 2 * ld, ws, None)


BAD_CACHE = [dict(k=0), dict(v_scale=0), dict(batch=0), dict(batch=32768), dict(heads=0), dict(rows=0),
             dict(rows=1 << 31), dict(dim=72), dict(dim=272), dict(dim=0), dict(block=8), dict(block=48),
             dict(k=(1 << 20) + 8), dict(v=(1 << 21) + 1), dict(k_scale=(1 << 22) + 2), dict(bs=4 * 100 * 64 + 8),
             dict(hs=8), dict(hs=0), dict(bs=0), dict(bs=-1024), dict(rs=48), dict(rs=72), dict(shs=3), dict(sbs=0),
             dict(rows=(1 << 31) - 255), dict(hs=64, bs=400 * 64), dict(bs=2 * 100 * 64), dict(sbs=8), dict(shs=4, sbs=4)]


@pytest.mark.parametrize("fn", ["append", "read", "attn"])
@pytest.mark.parametrize("bad", BAD_CACHE, ids=str)
def test_bad_cache_is_refused_before_any_device_call(fn, bad):
    assert call(fn, desc(**bad)) < 0
    assert "onpu_kv8_" + fn in L.last_error()


@pytest.mark.parametrize("fn", ["append", "read", "attn"])
def test_null_cache_pos_and_bad_token_counts(fn):
    assert call(fn, None) < 0 and "onpu_kv8_" + fn in L.last_error()
    assert call(fn, desc(), pos=None) < 0 and "onpu_kv8_" + fn in L.last_error()
    assert call(fn, desc(), T=-1) < 0 and "token count" in L.last_error()
    assert call(fn, desc(), T=1 << 31) < 0 and "token count" in L.last_error()


BAD_CALL = [("append", dict(rows=(1 << 24) + 8), "k"), ("append", dict(ld=255), "k"), ("append", dict(ld=252), "k"),
            ("append", dict(ld=258, bf16=0), "k"), ("append", dict(rows=None), "k"), ("read", dict(ld=128), "k"),
            ("read", dict(rows=(1 << 24) + 2, bf16=0), "k"), ("attn", dict(rows=(1 << 24) + 4), "q"),
            ("attn", dict(out=(1 << 24) + 8), "out"), ("attn", dict(out=None), "out"), ("attn", dict(ld=250), "q"),
            ("attn", dict(ws=None), "ws"), ("attn", dict(ws=(1 << 26) + 8), "ws"), ("attn", dict(Hq=6), "Hq"),
            ("attn", dict(Hq=0), "Hq"), ("attn", dict(Hq=68), "Hq"), ("attn", dict(Hq=-8), "Hq")]


@pytest.mark.parametrize("fn,bad,what", BAD_CALL, ids=str)
def test_bad_rows_heads_and_workspace_are_refused(fn, bad, what):
    assert call(fn, desc(), **bad) < 0
    assert what in L.last_error() and "onpu_kv8_" + fn in L.last_error()


def test_append_refuses_one_buffer_for_both():
    assert call("append", desc(v=GOOD["k"])) < 0 and "same" in L.last_error()
    assert call("append", desc(v_scale=GOOD["k_scale"])) < 0 and "same" in L.last_error()


def test_no_tokens_is_no_call():
    for fn in ("append", "read", "attn"):
        assert call(fn, desc(), T=0, rows=None, out=None, ws=None) == 0


def test_workspace_query_refuses_what_the_call_refuses():
    for d, Hq in ((desc(dim=24), 8), (desc(), 6)):
        assert L.load().onpu_kv8_attn_ws(C.addressof(d), Hq, 1, 1) < 0
        assert "onpu_kv8_attn_ws" in L.last_error()


def test_wrapper_refuses_cpu_tensors():
    k = torch.zeros(1, 1, 32, 64, dtype=torch.int8)
    s = torch.zeros(1, 1, 1)
    with pytest.raises(L.OnpuError):
        kv8.KVCache8.from_tensors(k, k.clone(), s, s.clone())


# ---------------------------------------------------------------- the oracle by hand
def test_oracle_scale_grows_and_older_rows_follow():
    codes, scales = np.zeros((1, 1, 32, 16), np.int8), np.zeros((1, 1, 2), np.float32)
    x = np.zeros((1, 2, 1, 16), np.float32)
    x[0, 0, 0, :3] = 127, 63.5, -1          # scale 1: 63.5 ties to even 64
    x[0, 1, 0, :2] = 254, -3                # scale 2: -1.5 ties to -2; the first row re-rounds to 64, 32, -0
    O.kv8_append(codes, scales, x[:, :1], [3], [1], 16)
    assert scales[0, 0, 0] == 1 and codes[0, 0, 3, :3].tolist() == [127, 64, -1]
    O.kv8_append(codes, scales, x[:, 1:], [4], [1], 16)
    assert scales[0, 0, 0] == 2 and codes[0, 0, 3, :3].tolist() == [64, 32, 0] and codes[0, 0, 4, :2].tolist() == [127, -2]
    O.kv8_append(codes, scales, x[:, :1], [0], [1], 16)          # a block's first row starts it anew
    assert scales[0, 0, 0] == 1
    x[0, 0, 0, 5] = np.inf
    O.kv8_append(codes, scales, x[:, :1], [17], [1], 16)
    assert np.isnan(scales[0, 0, 1]) and not codes[0, 0, 17].any()


def test_oracle_attention_matches_attn_step():
    """On one sequence and one token the definition is attn_step's over the cache's values."""
    rng = np.random.default_rng(3)
    codes = rng.integers(-127, 128, (1, 2, 50, 32)).astype(np.int8)
    scales = rng.uniform(0.01, 0.03, (1, 2, 4)).astype(np.float32)
    K = O.kv8_values(codes, scales, 16)
    V = K[:, ::-1]
    q = rng.normal(size=(1, 1, 6, 32)).astype(np.float32)
    mask = np.where(rng.random((1, 1, 50)) < 0.2, -np.inf, 0).astype(np.float32)
    sinks = rng.normal(size=6).astype(np.float32)
    got, _ = O.kv8_attn(q, K, V, [49], [1], mask, sinks)
    ref = O.attn_step(q[0, 0], K[0], V[0], mask[0, 0], sinks)
    assert np.abs(got[0, 0] - ref).max() < 1e-6      # attn_step rounds its result to fp32
