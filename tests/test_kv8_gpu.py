"""The 8-bit KV cache on the GPU (kv8.cu, kv8_attn.cu) against the float64 oracle (oracle.kv8_*).

Writing is exact: codes and scales equal the oracle's bit for bit. Reading is one fp32 product (half a
step, 2^-24) and, for bf16, one more rounding (2^-8 of the value). Attention's bound, with big the largest
sum |q_d k_d| scale over a query's rows, n its rows and vmax the largest value: a score is off by big *
(D 2^-23 + 2^-21) (sums of D exact products in fp32, possibly truncated; the query's rounding to 22 bits or more)
and e^x by that plus 2^-20 of itself; both enter the numerator and the sum, and adding n terms in
16-row steps costs (n / 16 + 64) 2^-23. bf16 calls round e^x to 11 bits (2^-11 at most) and the output
(2^-8 of it)."""
import ctypes as C

import numpy as np
import pytest
import torch

from opennpu_b200 import libonpu as L
from opennpu_b200.kv8 import KVCache8
from oracle import oracle as O

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def i32(a):
    return torch.tensor(list(a), dtype=torch.int32, device="cuda")


def status():
    torch.cuda.synchronize()
    return L.load().onpu_check_device()


def rand_cache(rng, B, H, S, D, block, spread=0.02):
    """codes and scales as numpy (k, v, ks, vs)"""
    codes = [np.clip(np.rint(rng.normal(size=(B, H, S, D)) * 36), -127, 127).astype(np.int8) for _ in range(2)]
    scales = [rng.uniform(0.018, 0.018 + spread, (B, H, -(-S // block))).astype(np.float32) for _ in range(2)]
    return (*codes, *scales)


def rand_rows(rng, shape, dtype):
    """numpy fp32 values that dtype holds exactly, and the CUDA tensor"""
    x = rng.normal(size=shape).astype(np.float32)
    t = torch.from_numpy(x).to(DT[dtype])
    return t.float().numpy(), t.cuda()


def bind(cache, block):
    return KVCache8.from_tensors(*(dev(a) for a in cache), block)


def check_attn(got, q, cache, block, pos, cnt, mask=None, sinks=None, scale=None, bf16=False):
    K, V = O.kv8_values(cache[0], cache[2], block), O.kv8_values(cache[1], cache[3], block)
    ref, big = O.kv8_attn(q, K, V, pos, cnt, mask, sinks, scale)
    D = q.shape[3]
    got = got.double().cpu().numpy()
    for b in range(q.shape[0]):
        for i in range(int(cnt[b])):
            n = int(pos[b]) + i + 1
            vmax = np.abs(V[b, :, :n]).max()
            tol = vmax * (2 * (big[b, i][:, None] * (D * 2.0 ** -23 + 2.0 ** -21) + 2.0 ** -20) + (n / 16 + 64) * 2.0 ** -23 +
                          (2.0 ** -11 if bf16 else 0)) + np.abs(ref[b, i]) * (2.0 ** -8 if bf16 else 2.0 ** -23)
            err = np.abs(got[b, i] - ref[b, i])
            assert (err <= tol).all(), (b, i, float(err.max()), float(tol.min()))
    return ref


# ---------------------------------------------------------------- writing
@pytest.mark.parametrize("B,T,H,D,S,block,dtype,pos,cnt", [
    (1, 1, 1, 16, 1, 16, "fp32", [0], None),               # the smallest cache
    (1, 1, 8, 128, 100, 32, "bf16", [57], None),
    (5, 1, 3, 64, 64, 32, "bf16", [0, 31, 32, 33, 63], None),
    (3, 7, 2, 80, 90, 16, "fp32", [0, 13, 83], [7, 5, 7]),
    (2, 33, 2, 256, 130, 64, "fp32", [1, 97], [33, 32]),
    (4, 200, 4, 128, 300, 32, "bf16", [0, 5, 31, 100], [200, 1, 0, 199]),
    (2, 130, 1, 112, 200, 64, "bf16", [63, 64], None),
    (1, 100, 2, 256, 128, 64, "bf16", [28], None),
    (2, 16, 2, 192, 40, 16, "fp32", [8, 24], None),
])
def test_append_is_exact(B, T, H, D, S, block, dtype, pos, cnt):
    rng = np.random.default_rng(B * 1000 + T + D)
    cache = rand_cache(rng, B, H, S, D, block, 0.01)
    c = bind(cache, block)
    k, kt = rand_rows(rng, (B, T, H, D), dtype)
    v, vt = rand_rows(rng, (B, T, H, D), dtype)
    c.append(kt, vt, i32(pos), None if cnt is None else i32(cnt))
    n = [T] * B if cnt is None else cnt
    O.kv8_append(cache[0], cache[2], k, pos, n, block)
    O.kv8_append(cache[1], cache[3], v, pos, n, block)
    assert status() == 0
    for got, ref in zip((c.k, c.v, c.k_scale, c.v_scale), cache):
        assert np.array_equal(got.cpu().numpy(), ref)


@pytest.mark.parametrize("block", [16, 32, 64])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_tokens_appended_one_by_one_with_growing_values(block, dtype):
    """Every append re-rounds its block: the chain of roundings is the definition's."""
    B, H, D, S = 2, 2, 64, 100
    rng = np.random.default_rng(block)
    cache = [np.zeros((B, H, S, D), np.int8), np.zeros((B, H, S, D), np.int8)] + \
            [np.zeros((B, H, -(-S // block)), np.float32) for _ in range(2)]
    c = KVCache8(B, H, S, D, block)
    for step in range(70):
        pos = [step, step + 20]
        k, kt = rand_rows(rng, (B, 1, H, D), dtype)
        k, kt = k * 2.0 ** (step % 9 - 4), kt * 2.0 ** (step % 9 - 4)
        c.append(kt, kt, i32(pos))
        O.kv8_append(cache[0], cache[2], k, pos, [1, 1], block)
    torch.cuda.synchronize()
    assert np.array_equal(c.k.cpu().numpy(), cache[0]) and np.array_equal(c.k_scale.cpu().numpy(), cache[2])
    assert np.array_equal(c.v.cpu().numpy(), cache[0]) and np.array_equal(c.v_scale.cpu().numpy(), cache[2])


def test_append_ties_extremes_and_values_that_are_not_finite():
    """Halves of a step (ties to even), zeros, values whose scale is subnormal or huge; infinities and
    NaN poison their own block and head only, until the block is begun again."""
    H, D, S, block = 8, 64, 64, 16
    x = np.zeros((1, S, H, D), np.float32)
    j = np.arange(S)[:, None]
    x[0, :, 0] = (j * 64 + np.arange(D)) % 255 / 2 - 63.5
    x[0, ::block, 0, 0] = 127                            # scale 1: halves are ties
    x[0, :, 1] = 0
    x[0, :, 2] = np.float32(1e-44) * (1 + np.arange(D) % 3)
    x[0, :, 3] = np.linspace(-3.4e38, 3.4e38, D, dtype=np.float32)
    x[0, :, 4] = np.float32(2.0 ** -126) * np.linspace(-1, 1, D, dtype=np.float32)
    x[0, :, 5] = np.arange(D) - 32
    x[0, 3, 5, 7] = np.inf
    x[0, 40, 5, 0] = np.nan
    x[0, 63, 5, 63] = -np.inf
    x[0, :, 6] = np.random.default_rng(0).normal(size=(S, D)) * np.float32(1e30)
    x[0, :, 7] = np.float32(0.1) * (np.arange(D) - 31)
    ref = [np.zeros((1, H, S, D), np.int8), np.zeros((1, H, S // block), np.float32)]
    with np.errstate(all="ignore"):
        O.kv8_append(ref[0], ref[1], x, [0], [S], block)
    c = KVCache8(1, H, S, D, block)
    c.append(dev(x), dev(x), i32([0]))
    torch.cuda.synchronize()
    assert np.array_equal(c.k_scale.cpu().numpy(), ref[1], equal_nan=True)
    assert np.array_equal(c.k.cpu().numpy(), ref[0])
    assert np.isnan(ref[1][0, 5]).tolist() == [True, False, True, True]
    k, _ = c.read(i32([0]), tokens=S, dtype=torch.float32)
    assert torch.isnan(k[0, :16, 5]).all() and not torch.isnan(k[0, :, :5]).any()
    one = torch.ones(1, 1, H, D, device="cuda")
    c.append(one, one, i32([4]))                         # the NaN stays while the block does
    assert torch.isnan(c.k_scale[0, 5, 0])
    c.append(one, one, i32([0]))                         # and goes with its first row
    assert c.k_scale[0, 5, 0].item() == np.float32(1 / 127)


def test_rows_behind_a_sequence_and_other_sequences_stay():
    B, H, D, S, block = 4, 2, 64, 64, 32
    rng = np.random.default_rng(5)
    cache = rand_cache(rng, B, H, S, D, block)
    c = bind(cache, block)
    x = torch.full((B, 8, H, D), 50.0, device="cuda")
    x[1, 3:] = float("nan")                              # padding is never read
    x[2] = float("nan")
    c.append(x, x, i32([10, 10, 10, 40]), i32([8, 3, 0, 8]))
    k = c.k.cpu().numpy()
    assert np.array_equal(k[2], cache[0][2]) and np.array_equal(c.v_scale.cpu().numpy()[2], cache[3][2])
    assert np.array_equal(k[0, :, 18:], cache[0][0, :, 18:]) and np.array_equal(k[1, :, 13:], cache[0][1, :, 13:])
    assert np.array_equal(k[3, :, :32], cache[0][3, :, :32]) and (k[1, :, 10:13] == 127).all()
    assert status() == 0
    out = [torch.full((B, 8, H, D), 7.0, device="cuda") for _ in range(2)]
    c.read(i32([10, 10, 10, 40]), i32([8, 3, 0, 8]), out=out)
    q = torch.randn(B, 8, 4, D, device="cuda")
    y = torch.full_like(q, 7.0)
    c.attn(q, i32([10, 10, 10, 40]), i32([8, 3, 0, 8]), out=y)
    for t in (*out, y):
        assert (t[1, 3:] == 7).all() and (t[2] == 7).all() and not (t[0] == 7).any() and torch.isfinite(t).all()


# ---------------------------------------------------------------- reading
@pytest.mark.parametrize("B,T,H,D,S,block,dtype,pos,cnt", [
    (1, 1, 1, 16, 1, 16, "fp32", [0], None), (2, 37, 3, 80, 50, 16, "bf16", [13, 0], [37, 20]),
    (3, 64, 2, 256, 65, 64, "fp32", [1, 0, 0], [64, 64, 0]), (2, 500, 8, 128, 600, 32, "bf16", [99, 100], None)])
def test_read_back(B, T, H, D, S, block, dtype, pos, cnt):
    rng = np.random.default_rng(T)
    cache = rand_cache(rng, B, H, S, D, block)
    c = bind(cache, block)
    k, v = c.read(i32(pos), None if cnt is None else i32(cnt), tokens=T, dtype=DT[dtype])
    for got, codes, scales in ((k, cache[0], cache[2]), (v, cache[1], cache[3])):
        ref = O.kv8_values(codes, scales, block)
        for b in range(B):
            n = T if cnt is None else cnt[b]
            r = ref[b, :, pos[b]:pos[b] + n].transpose(1, 0, 2)
            g = got[b, :n].double().cpu().numpy()
            assert (np.abs(g - r) <= np.abs(r) * (2.0 ** -24 + (2.0 ** -8 if dtype == "bf16" else 0))).all()


# ---------------------------------------------------------------- attention
ATTN = [  # B, T, Hq, H, D, S, block, dtype, pos, cnt
    (1, 1, 1, 1, 16, 1, 16, "fp32", [0], None),
    (1, 1, 8, 2, 64, 40, 32, "fp32", [0], None),              # one row
    (1, 1, 32, 8, 128, 700, 32, "fp32", [699], None),
    (1, 1, 32, 8, 128, 700, 32, "bf16", [640], None),
    (3, 1, 16, 1, 128, 333, 64, "bf16", [332, 0, 64], None),     # 16 query heads on one kv head
    (2, 1, 7, 7, 80, 150, 16, "fp32", [149, 15], None),
    (2, 1, 12, 3, 192, 150, 32, "bf16", [31, 128], None),
    (2, 1, 8, 2, 256, 1000, 64, "fp32", [999, 500], None),
    (1, 1, 5, 1, 112, 97, 16, "bf16", [96], None),
    (2, 5, 16, 2, 64, 220, 32, "fp32", [200, 11], [5, 3]),       # draft tokens, a padded batch
    (2, 16, 24, 2, 96, 130, 16, "fp32", [0, 100], [16, 9]),
    (4, 3, 4, 4, 128, 90, 32, "bf16", [0, 30, 31, 87], [3, 0, 1, 3]),
    (2, 40, 8, 2, 128, 400, 32, "bf16", [0, 333], [40, 37]),     # prompt chunks
    (1, 130, 10, 2, 128, 500, 32, "bf16", [250], None),
    (1, 77, 6, 2, 256, 200, 64, "bf16", [100], None),
    (2, 65, 3, 3, 64, 300, 16, "bf16", [0, 200], [65, 64]),
    (1, 19, 16, 1, 80, 150, 32, "bf16", [128], None),
    (1, 50, 4, 2, 128, 128, 32, "fp32", [70], None),
]


@pytest.mark.parametrize("extra", ["plain", "mask+sinks"])
@pytest.mark.parametrize("case", ATTN, ids=str)
def test_attention(case, extra):
    B, T, Hq, H, D, S, block, dtype, pos, cnt = case
    rng = np.random.default_rng(S * 7 + T)
    cache = rand_cache(rng, B, H, S, D, block)
    c = bind(cache, block)
    q, qt = rand_rows(rng, (B, T, Hq, D), dtype)
    mask = sinks = None
    if extra != "plain":
        mask = np.where(rng.random((B, T, S)) < 0.3, -np.inf, rng.normal(size=(B, T, S))).astype(np.float32)
        sinks = rng.normal(size=Hq).astype(np.float32)
    y = c.attn(qt, i32(pos), None if cnt is None else i32(cnt), None if mask is None else dev(mask),
               None if sinks is None else dev(sinks))
    check_attn(y, q, cache, block, pos, [T] * B if cnt is None else cnt, mask, sinks, bf16=dtype == "bf16")
    assert status() == 0
    assert torch.equal(y[0, :1], c.attn(qt, i32(pos), None if cnt is None else i32(cnt),
                                        None if mask is None else dev(mask), None if sinks is None else dev(sinks))[0, :1])


@pytest.mark.parametrize("T,dtype", [(1, "fp32"), (1, "bf16"), (6, "fp32"), (64, "bf16")])
def test_masks_that_leave_nothing_or_little(T, dtype):
    """Query 0 masked everywhere (zeros, sinks or not), query 1 where there is one left a single row, runs that blank
    whole stretches, and masks of the lowest finite value, which weigh rows equally where all have it."""
    B, Hq, H, D, S, block = 2, 8, 2, 128, 900, 32
    rng = np.random.default_rng(T)
    cache = rand_cache(rng, B, H, S, D, block)
    c = bind(cache, block)
    q, qt = rand_rows(rng, (B, T, Hq, D), dtype)
    pos, cnt = [S - T, 300], [T, T]
    low = np.finfo(np.float32).min
    mask = np.zeros((B, T, S), np.float32)
    mask[0, 0] = -np.inf
    mask[1, 0] = low
    if T > 1:
        mask[0, 1] = -np.inf
        mask[0, 1, 17] = 0.5
        mask[0, 2:, :600] = -np.inf
        mask[1, 1:, 100:250] = low
    for sinks in (None, rng.normal(size=Hq).astype(np.float32)):
        y = c.attn(qt, i32(pos), None, dev(mask), None if sinks is None else dev(sinks))
        assert (y[0, 0] == 0).all()
        check_attn(y, q, cache, block, pos, cnt, mask, sinks, bf16=dtype == "bf16")


@pytest.mark.parametrize("T,dtype", [(1, "fp32"), (3, "bf16"), (64, "bf16")])
def test_what_masked_rows_hold_does_not_matter(T, dtype):
    """Blocks whose scales are NaN, masked with -inf, and NaN scales behind the sequences; unmasked
    they make the queries that see them NaN, and only those."""
    B, Hq, H, D, S, block = 2, 6, 2, 64, 320, 32
    rng = np.random.default_rng(T)
    cache = rand_cache(rng, B, H, S, D, block)
    pos, cnt = [96 - T, 200 - T], [T, T]
    for s in cache[2:]:
        s[0, :, 3:] = np.nan
        s[1, :, 7:] = np.nan
    c = bind(cache, block)
    q, qt = rand_rows(rng, (B, T, Hq, D), dtype)
    y = c.attn(qt, i32(pos))
    check_attn(y, q, tuple(np.nan_to_num(a) for a in cache), block, pos, cnt, bf16=dtype == "bf16")
    cache[2][:, :, 1] = np.nan
    cache[3][:, :, 1] = np.nan
    mask = np.zeros((B, T, S), np.float32)
    mask[:, :, 32:64] = -np.inf
    c = bind(cache, block)
    y = c.attn(qt, i32(pos), None, dev(mask))
    check_attn(y, q, tuple(np.nan_to_num(a) for a in cache), block, pos, cnt, mask, bf16=dtype == "bf16")
    mask[0, 0, 40] = 0
    y = c.attn(qt, i32(pos), None, dev(mask))
    nan = torch.isnan(y).all(-1).all(-1).cpu()               # query 0 of sequence 0, where it stands behind row 40
    assert nan[0].tolist() == [pos[0] >= 40] + [False] * (T - 1) and not nan[1].any()
    assert torch.isfinite(y[1]).all() and torch.isfinite(y[0, 1:]).all()


@pytest.mark.parametrize("T,dtype", [(1, "fp32"), (1, "bf16"), (3, "fp32"), (64, "bf16"), (40, "fp32")])
@pytest.mark.parametrize("power", [121, -100])
def test_queries_and_scales_at_the_ends_of_the_range(T, dtype, power):
    """Queries times 2^power over keys times 2^-power give the scores they give at 1; values near 2^100 and
    2^-100; a head of zero queries weighs rows equally; a query that is not finite gives NaN, alone."""
    B, Hq, H, D, S, block = 2, 6, 2, 64, 150, 32
    rng = np.random.default_rng(T)
    cache = rand_cache(rng, B, H, S, D, block)
    cache[2][:] = cache[2] * np.float32(2.0 ** -power)
    cache[3][:] = cache[3] * np.float32(2.0 ** (100 if power > 0 else -100))
    q, qt = rand_rows(rng, (B, T, Hq, D), dtype)
    q, qt = q * np.float32(2.0 ** power), qt * 2.0 ** power
    q[:, :, 2], qt[:, :, 2] = 0, 0
    c = bind(cache, block)
    pos, cnt = [S - T, 20], [T, T]
    y = c.attn(qt, i32(pos))
    check_attn(y, q, cache, block, pos, cnt, bf16=dtype == "bf16")
    qt[0, T - 1, 1, 5] = float("inf")
    qt[1, 0, 4, 0] = float("nan")
    z = c.attn(qt, i32(pos))
    same = torch.ones(B, T, Hq, dtype=torch.bool)
    same[0, T - 1, 1] = same[1, 0, 4] = False
    assert torch.equal(z[same], y[same]) and torch.isnan(z[~same]).all()


@pytest.mark.parametrize("T,dtype", [(1, "fp32"), (1, "bf16"), (3, "fp32"), (70, "fp32"), (70, "bf16")])
def test_queries_whose_largest_value_is_all_ones(T, dtype):
    """The largest significand (2 - 2^-23, bf16 2 - 2^-7) of either sign: its rounded digits must not wrap."""
    rng = np.random.default_rng(T)
    cache = rand_cache(rng, 1, 2, 150, 64, 32)
    c = bind(cache, 32)
    q, _ = rand_rows(rng, (1, T, 4, 64), dtype)
    top = np.float32(2 - (2.0 ** -23 if dtype == "fp32" else 2.0 ** -7)) * 4
    q = np.clip(q, -7, 7)
    q[..., 3], q[..., 40] = top, -top
    y = c.attn(torch.from_numpy(q).to(DT[dtype]).cuda(), i32([150 - T]))
    check_attn(y, q, cache, 32, [150 - T], [T], bf16=dtype == "bf16")


def test_negative_and_zero_scale():
    B, Hq, H, D, S = 1, 4, 2, 64, 200
    rng = np.random.default_rng(2)
    cache = rand_cache(rng, B, H, S, D, 32)
    c = bind(cache, 32)
    for T, dtype in ((1, "fp32"), (1, "bf16"), (80, "bf16")):
        q, qt = rand_rows(rng, (B, T, Hq, D), dtype)
        for scale in (-0.3, 0.0):
            y = c.attn(qt, i32([S - T]), scale=scale)
            check_attn(y, q, cache, 32, [S - T], [T], scale=scale, bf16=dtype == "bf16")


def test_scores_that_grow_along_the_rows():
    """Later rows outweigh all earlier ones again and again: the reference moves in every step, by a little
    and by more than fp16 spans; and a value scale that grows past the weights' range."""
    B, Hq, H, D, S, block = 1, 8, 2, 128, 1500, 16
    rng = np.random.default_rng(4)
    cache = list(rand_cache(rng, B, H, S, D, block))
    for steep in (0.02, 0.6):
        cache[0][...] = 100
        cache[2][...] = (steep * np.arange(cache[2].shape[2]) / (100 * D) * D ** 0.5).astype(np.float32)
        cache[3][...] = (2.0 ** (np.arange(cache[3].shape[2]) // 4 - 12)).astype(np.float32)
        c = bind(tuple(cache), block)
        for T, dtype in ((1, "fp32"), (1, "bf16"), (60, "bf16"), (40, "fp32")):
            q = np.ones((B, T, Hq, D), np.float32)
            y = c.attn(torch.from_numpy(q).to(DT[dtype]).cuda(), i32([S - T]))
            check_attn(y, q, cache, block, [S - T], [T], bf16=dtype == "bf16")


def test_strides_slices_and_broadcast_masks():
    """A cache kept [B, rows, heads, dim], sequences sliced out of a larger cache, q / k / v as slices of
    fused projection rows, masks broadcast over sequences and tokens, a scale and an out of the caller's."""
    B, T, Hq, H, D, S, block = 2, 4, 6, 2, 64, 96, 16
    rng = np.random.default_rng(11)
    cache = rand_cache(rng, B, H, S, D, block)
    nb = S // block
    big = [torch.zeros(B + 3, S, H, D, dtype=torch.int8, device="cuda")[2:2 + B].permute(0, 2, 1, 3) for _ in range(2)]
    sc = [torch.zeros(B + 3, H, nb + 5, device="cuda")[2:2 + B, :, :nb] for _ in range(2)]
    for t, a in zip(big + sc, cache):
        t.copy_(dev(a))
    c = KVCache8.from_tensors(*big, *sc, block)
    fused = torch.randn(B, T, Hq + 2 * H, D, device="cuda")
    q, k, v = fused.split([Hq, H, H], 2)
    pos, cnt = [20, 92], [4, 4]
    c.append(k, v, i32(pos))
    for i, x in ((0, k), (1, v)):
        O.kv8_append(cache[i], cache[i + 2], x.cpu().numpy(), pos, cnt, block)
    for got, ref in zip((c.k, c.v, c.k_scale, c.v_scale), cache):
        assert np.array_equal(got.cpu().numpy(), ref)
    for shape in ((1, 1, S), (B, 1, S), (1, T, S), (B, T, S)):
        mask = np.where(rng.random(shape) < 0.3, -np.inf, 0).astype(np.float32)
        out = torch.zeros(B, T, Hq + 1, D, device="cuda")[:, :, :Hq]
        y = c.attn(q, i32(pos), None, dev(mask), scale=0.2, out=out)
        assert y.data_ptr() == out.data_ptr()
        check_attn(y, q.cpu().numpy(), cache, block, pos, cnt, np.broadcast_to(mask, (B, T, S)), scale=0.2)
    kr, vr = c.read(i32(pos), tokens=T, dtype=torch.float32)
    ref = O.kv8_values(cache[1], cache[3], block)
    assert np.abs(vr[1].cpu().numpy() - ref[1, :, 92:96].transpose(1, 0, 2)).max() <= 2.0 ** -24 * np.abs(ref).max()


def test_one_query_head_per_sequence_in_a_large_ragged_batch():
    """More sequences than the grid has CTAs, most of them short, some empty."""
    B, H, D, S, block = 700, 1, 64, 40, 16
    rng = np.random.default_rng(1)
    cache = rand_cache(rng, B, H, S, D, block)
    c = bind(cache, block)
    q, qt = rand_rows(rng, (B, 1, 2, D), "fp32")
    pos = rng.integers(0, S, B)
    cnt = (np.arange(B) % 5 != 0).astype(int)
    y = c.attn(qt, i32(pos), i32(cnt))
    check_attn(y, q, cache, block, pos, cnt)


def test_long_cache_offsets_pass_32_bits():
    """Rows beyond 2^31 codes and 2^31 bytes of a head: written, read back, and weighed alone by a mask."""
    S, D, block = (1 << 24) + 70, 256, 64
    c = KVCache8(1, 1, S, D, block)
    x = torch.randn(1, 40, 1, D, device="cuda")
    pos = i32([S - 40])
    c.append(x, x.flip(1), pos)
    ref = [np.zeros((1, 1, 128, D), np.int8), np.zeros((1, 1, 2), np.float32)]
    first = (S - 40) // block * block
    O.kv8_append(ref[0], ref[1], x.cpu().numpy(), [S - 40 - first], [40], block)
    n = S - first
    assert np.array_equal(c.k[0, 0, first:].cpu().numpy(), ref[0][0, 0, :n])
    k, v = c.read(pos, tokens=40, dtype=torch.float32)
    got = c.k[0, 0, -40:].float() * c.k_scale[0, 0, (torch.arange(S - 40, S, device="cuda") // block)][:, None]
    assert torch.equal(k[0, :, 0], got)
    mask = torch.full((1, 1, S), float("-inf"), device="cuda")
    mask[0, 0, S - 3] = 0
    for dtype in (torch.float32, torch.bfloat16):
        y = c.attn(x[:, :1].to(dtype).contiguous(), i32([S - 1]), mask=mask)
        assert (y[0, 0, 0].float() - v[0, 37, 0]).abs().max() <= v[0, 37, 0].abs().max() * 2.0 ** -8
    y = c.attn(x[:, -40:].to(torch.bfloat16).contiguous(), pos, mask=mask)
    assert (y[0, :37] == 0).all() and (y[0, 37:, 0].float() - v[0, 37, 0]).abs().max() <= v[0, 37, 0].abs().max() * 2.0 ** -8


# ---------------------------------------------------------------- as a program uses them
def test_places_outside_the_cache_are_skipped_and_reported():
    B, H, D, S = 5, 2, 64, 48
    c = KVCache8(B, H, S, D, 16)
    x = torch.ones(B, 4, H, D, device="cuda")
    pos, cnt = i32([0, 45, -1, 3, 0]), i32([4, 4, 2, 5, -1])
    y, out = torch.full_like(x, 7), [torch.full_like(x, 7) for _ in range(2)]
    for call in (lambda: c.append(x, x, pos, cnt), lambda: c.attn(x, pos, cnt, out=y),
                 lambda: c.read(pos, cnt, out=out)):
        call()
        assert status() == -2 and "8-bit KV cache" in L.last_error()
        assert status() == 0
    assert (c.k[0, :, :4] == 127).all() and not c.k[1:].any() and not c.v_scale[1:].any()
    for t in (y, *out):
        assert (t[0] != 7).all() and (t[1:] == 7).all()


def test_wrapper_refusals():
    c = KVCache8(2, 2, 32, 64, 16)
    x, pos = torch.zeros(2, 3, 2, 64, device="cuda"), i32([0, 0])
    bad = [lambda: c.append(x, x, pos.long()), lambda: c.append(x, x, pos[:1]), lambda: c.append(x, x.bfloat16(), pos),
           lambda: c.append(x, x[:, :2], pos), lambda: c.append(x.half(), x.half(), pos),
           lambda: c.append(x[:, :, :1], x[:, :, :1], pos), lambda: c.append(x.cpu(), x.cpu(), pos),
           lambda: c.append(x, x, pos.cpu()), lambda: c.append(x.transpose(1, 2), x.transpose(1, 2), pos),
           lambda: c.append(x[..., :32], x[..., :32], pos), lambda: c.read(pos),
           lambda: c.attn(torch.zeros(2, 3, 3, 64, device="cuda"), pos),
           lambda: c.attn(torch.zeros(2, 3, 34, 64, device="cuda"), pos),
           lambda: c.attn(x, pos, mask=torch.zeros(2, 3, 31, device="cuda")),
           lambda: c.attn(x, pos, mask=torch.zeros(2, 2, 32, device="cuda")),
           lambda: c.attn(x, pos, mask=torch.zeros(2, 3, 32, device="cuda", dtype=torch.bool)),
           lambda: c.attn(x, pos, sinks=torch.zeros(3, device="cuda")),
           lambda: c.attn(x, pos, out=torch.zeros(2, 3, 2, 64, device="cuda", dtype=torch.bfloat16)),
           lambda: c.attn(torch.zeros(2, 3, 129, device="cuda")[..., 1:].view(2, 3, 2, 64), pos),
           lambda: KVCache8(1, 1, 32, 72), lambda: KVCache8(1, 1, 32, 64, block=8),
           lambda: KVCache8.from_tensors(c.k, c.v[:, :, :16], c.k_scale, c.v_scale, 16),
           lambda: KVCache8.from_tensors(c.k, c.v, c.k_scale[..., :1], c.v_scale[..., :1], 16),
           lambda: KVCache8.from_tensors(c.k.float(), c.v.float(), c.k_scale, c.v_scale, 16),
           lambda: KVCache8.from_tensors(c.k[:1].expand(2, -1, -1, -1), c.v[:1].expand(2, -1, -1, -1), c.k_scale,
                                         c.v_scale, 16).append(x, x, pos)]
    for i, f in enumerate(bad):
        with pytest.raises(L.OnpuError):
            f()
            pytest.fail(f"call {i} was taken")
    assert status() == 0


def decode_step(c, x, pos, out):
    """append, then attend: q / k / v as slices of one projection's rows"""
    H = c.heads
    q, k, v = x.split([x.shape[2] - 2 * H, H, H], 2)
    c.append(k, v, pos)
    return c.attn(q, pos, out=out)


def test_decode_loop_in_a_replayed_graph_matches_eager_calls():
    """A decode step captured once and replayed while pos grows on the device: the caches and outputs of
    every step equal the eager calls', across block borders."""
    B, Hq, H, D, S, block = 3, 8, 2, 128, 80, 16
    g = torch.Generator(device="cuda").manual_seed(0)
    xs = torch.randn(60, B, 1, Hq + 2 * H, D, device="cuda", generator=g).to(torch.bfloat16)
    eager, graphed = KVCache8(B, H, S, D, block), KVCache8(B, H, S, D, block)
    x, pos, out = xs[0].clone(), i32([0, 7, 19]), torch.zeros(B, 1, Hq, D, device="cuda", dtype=torch.bfloat16)
    decode_step(graphed, x, pos, out)                        # warm-up; row pos is written again below
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        decode_step(graphed, x, pos, out)
    for i in range(60):
        x.copy_(xs[i])
        graph.replay()
        y = decode_step(eager, xs[i], pos, torch.empty_like(out))
        assert torch.equal(y, out) and torch.isfinite(y).all()
        pos += 1
    assert torch.equal(eager.k, graphed.k) and torch.equal(eager.v_scale, graphed.v_scale)
    assert status() == 0


FIRST_CALL_CAPTURED = """
import torch
from opennpu_b200 import libonpu as L
from opennpu_b200.kv8 import KVCache8
c = KVCache8(2, 2, 300, 128)
pos = torch.tensor([0, 90], dtype=torch.int32, device="cuda")
x = torch.randn(2, 100, 12, 128, device="cuda").bfloat16()
f = x[:, :3].float()
outs = []
def step():
    c.append(x[:, :, 8:10], x[:, :, 10:], pos)
    outs[:] = [c.attn(x[:, :, :8], pos), c.attn(f[:, :, :8], pos), *c.read(pos, tokens=100)]
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    step()
g.replay()
got = [t.clone() for t in outs]
step()
torch.cuda.synchronize()
assert all(torch.equal(a, b) and torch.isfinite(a).all() for a, b in zip(got, outs))
assert L.load().onpu_check_device() == 0
"""


def test_first_calls_may_be_captured():
    """In a fresh process: the first calls of every kind inside a capture, replayed, equal eager ones."""
    import subprocess
    import sys

    from tests.conftest import ROOT
    r = subprocess.run([sys.executable, "-c", FIRST_CALL_CAPTURED], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_calls_without_tokens():
    c = KVCache8(2, 2, 64, 64)
    x, pos = torch.zeros(2, 0, 2, 64, device="cuda"), i32([5, 64])
    c.append(x, x, pos)
    assert c.attn(x, pos).shape == x.shape and c.read(pos, tokens=0)[0].shape == x.shape
    y = torch.full((2, 3, 4, 64), 7.0, device="cuda")
    c.attn(y, pos, i32([0, 0]), out=y)
    assert (y == 7).all() and status() == 0


def test_two_graphs_and_an_eager_call_at_once_do_not_share_workspace():
    """Two captured calls replayed on two streams while a third runs eagerly on its own stream: each
    gives what it gives alone."""
    Hq, H, D, S = 32, 8, 128, 6000
    caches, qs, alone = [], [], []
    for i in range(3):
        rng = np.random.default_rng(i)
        caches.append(bind(rand_cache(rng, 1, H, S, D, 32), 32))
        qs.append(torch.randn(1, 1, Hq, D, device="cuda"))
        alone.append(caches[i].attn(qs[i], i32([S - 1])).clone())
    pos, graphs, outs = i32([S - 1]), [], []
    for i in range(2):
        gr = torch.cuda.CUDAGraph()
        outs.append(torch.empty_like(qs[i]))
        with torch.cuda.graph(gr):
            caches[i].attn(qs[i], pos, out=outs[i])
        graphs.append(gr)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        y = caches[2].attn(qs[2], pos, stream=streams[2])
    torch.cuda.synchronize()
    for got, ref in zip((*outs, y), alone):
        assert torch.equal(got, ref)


def test_prompt_then_decode_then_rejected_drafts():
    """The set as a program runs it: a prompt appended in chunks, decode steps, drafts of which some are
    rejected and written over; at the end the cache and the attention equal the oracle's."""
    B, Hq, H, D, S, block = 2, 8, 2, 64, 256, 32
    rng = np.random.default_rng(9)
    cache = [np.zeros((B, H, S, D), np.int8) for _ in range(2)] + [np.zeros((B, H, S // block), np.float32) for _ in range(2)]
    c = KVCache8(B, H, S, D, block)
    pos = np.array([0, 0])
    for T, keep in ((70, (70, 51)), (45, (45, 45)), (1, (1, 1)), (4, (2, 4)), (1, (1, 1)), (4, (1, 3)), (1, (1, 1))):
        x, xt = rand_rows(rng, (B, T, Hq + 2 * H, D), "bf16")
        q, k, v = xt.split([Hq, H, H], 2)
        cnt = np.array(keep) if T > 4 else np.array([T, T])
        c.append(k, v, i32(pos), i32(cnt))
        y = c.attn(q, i32(pos), i32(cnt))
        O.kv8_append(cache[0], cache[2], x[:, :, Hq:Hq + H], pos, cnt, block)
        O.kv8_append(cache[1], cache[3], x[:, :, Hq + H:], pos, cnt, block)
        check_attn(y, x[:, :, :Hq], cache, block, pos, cnt, bf16=True)
        pos = pos + np.array(keep)
    for got, ref in zip((c.k, c.v, c.k_scale, c.v_scale), cache):
        assert np.array_equal(got.cpu().numpy(), ref)
    assert status() == 0
