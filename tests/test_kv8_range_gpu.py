"""8-bit KV cache attention over long runs of rows and wide ranges of scales, against the definition in float64 for
chosen queries: every warp and CTA takes many steps, so sums are rescaled, stages come round, and rows that a query does
not see or hardly weighs stand beside those it does.

Bounds, with p_j the query's normalised weights, A_d = sum_j p_j |v_jd| (only rows that weigh anything count), n its rows and
big the largest sum |q_d k_d| scale over them:
  * a score is off by big (D 2^-23 + 2^-21) (D exact products summed in fp32, possibly cut off; 22 bits of the query), e^x by
    that plus 2^-20; numerator (A_d) and sum (|out|) both have it;
  * adding in 16-row steps, possibly cut off: (c / 16 + 128) 2^-23 A_d, c the rows that a CTA sums on its own, at most n: the
    list's 128-row units over at least 148 CTAs, two more for its ends; 128 for the parts joined;
  * fp16 weights: 2^-11 of each (A_d) for bf16 calls, 2^-21 for the two parts of fp32 calls. The largest stands at 2^5 or more, so
    those below 2^-19 of it (two parts: 2^-8) have parts under fp16's normal range, off by 2^-25, 2^-30 of the largest;
  * scales as powers of two in the exponent (bf16, many queries): logarithms up to 2^8 to 24 bits, a handful of them, 2^-13;
  * the output's own rounding, 2^-8 or 2^-24 of it."""
import numpy as np
import pytest
import torch

from opennpu_b200 import libonpu as L
from opennpu_b200.kv8 import KVCache8

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


def i32(a):
    return torch.tensor(list(a), dtype=torch.int32, device="cuda")


def status():
    torch.cuda.synchronize()
    return L.load().onpu_check_device()


def rand_cache(seed, B, H, S, D, block):
    """CUDA tensors k, v, k_scale, v_scale: values of about unit size"""
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = [torch.randn(B, H, S, D, device="cuda", generator=g).mul_(36).round_().clamp_(-127, 127).to(torch.int8)
             for _ in range(2)]
    scales = [torch.rand(B, H, -(-S // block), device="cuda", generator=g) * 0.02 + 0.018 for _ in range(2)]
    return [*codes, *scales]


def rand_q(seed, shape, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed + 1000)
    return torch.randn(shape, device="cuda", generator=g).to(DT[dtype])


def attend(cache, block, b, i, h, q, pos, mask=None, sinks=None):
    """One query's output in float64 and its bound."""
    k, v, ks, vs = cache
    (T, Hq, D), bf16 = q.shape[1:], q.dtype == torch.bfloat16
    g, n = h // (Hq // k.shape[1]), int(pos[b]) + i + 1
    rows = torch.arange(n, device=k.device)
    m = torch.zeros(n, dtype=torch.float64, device=k.device)
    if mask is not None:
        m = mask.expand(len(pos), T, k.shape[2])[b, i, :n].double()
        rows, m = rows[m > -np.inf], m[m > -np.inf]
    if not len(rows):
        return torch.zeros(D, dtype=torch.float64, device=k.device), 0.0
    s_k, s_v = (a[b, g].double()[rows // block] for a in (ks, vs))
    K, V, qv = k[b, g, rows].double(), v[b, g, rows].double(), q[b, i, h].double()
    x = (K @ qv) * s_k * D ** -0.5 + m
    big = float(((K.abs() @ qv.abs()) * s_k).max()) * D ** -0.5
    top = float(x.max()) if sinks is None else max(float(x.max()), float(sinks[h]))
    p = torch.exp(x - top)
    p /= p.sum() + (0.0 if sinks is None else float(torch.exp(sinks[h].double() - top)))
    w = p * s_v
    out, A = w @ V, w @ V.abs()
    d = big * (D * 2.0 ** -23 + 2.0 ** -21) + 2.0 ** -20
    alone = min(n, 128 * (k.shape[0] * k.shape[1] * -(-k.shape[2] // 128) / 148 + 2))
    tiny = int((w < w.max() * 2.0 ** (-19 if bf16 else -8)).sum())
    tol = A * (d + (alone / 16 + 128) * 2.0 ** -23 + (2.0 ** -11 + 2.0 ** -13 if bf16 else 2.0 ** -21)) + out.abs() * (
        d + (2.0 ** -8 if bf16 else 2.0 ** -23)) + 127 * w.max() * tiny * 2.0 ** -30
    return out, tol


def check(y, cache, block, queries, q, pos, mask=None, sinks=None):
    """The listed (b, i, h) of y against the definition."""
    for b, i, h in queries:
        out, tol = attend(cache, block, b, i, h, q, pos, mask, sinks)
        err = (y[b, i, h].double() - out).abs()
        assert bool((err <= tol).all()), (b, i, h, int(pos[b]) + i + 1, float(err.max()), float(out.abs().max()))


def sawtooth(n, tile_blocks, step, period):
    """Scales of n blocks: times 2^step from one run of tile_blocks to the next, back after `period` runs."""
    return 0.02 * 2.0 ** (step * (torch.arange(n, device="cuda") // tile_blocks % period)).float()


def some_queries(B, T, Hq, count=6):
    rng = np.random.default_rng(B + T + Hq)
    return [(0, 0, 0), (B - 1, T - 1, Hq - 1)] + [tuple(int(rng.integers(n)) for n in (B, T, Hq)) for _ in range(count)]


# ---------------------------------------------------------------- sums rescaled while products run
@pytest.mark.parametrize("D,T,step", [(128, 20, 3), (64, 32, 2), (112, 17, 5)])
def test_value_scales_that_grow_from_tile_to_tile_at_65_to_128_queries(D, T, step):
    """One query tile a kv head, several row tiles a CTA: the sums over the values are rescaled in most of them."""
    H, rep, S, block = 2, 4, 37900, 32
    cache = rand_cache(D, 1, H, S, D, block)
    cache[3][:] = sawtooth(cache[3].shape[2], 128 // block, step, 8)
    q = rand_q(D, (1, T, H * rep, D), "bf16")
    c = KVCache8.from_tensors(*cache, block)
    for _ in range(10):
        y = c.attn(q, i32([S - T]))
        check(y, cache, block, some_queries(1, T, H * rep, 1), q, [S - T])
    assert status() == 0


@pytest.mark.parametrize("D,T", [(128, 20), (64, 20), (128, 60)])
def test_scores_and_value_scales_that_grow_in_the_same_tile(D, T):
    """Both reasons to rescale a tile's sums at once: its scores pass the reference by more than 2^6, and its value scales the
    weights' range, in tile after tile of a CTA's run."""
    H, rep, S, block = 2, 4, 37900, 32
    cache = rand_cache(D + T, 1, H, S, D, block)
    cache[3][:] = sawtooth(cache[3].shape[2], 128 // block, 3, 8)
    cache[0][:] = (18 * (torch.arange(S, device="cuda") // 128 % 8))[:, None].to(torch.int8)
    q = rand_q(D, (1, T, H * rep, D), "bf16").abs()
    c = KVCache8.from_tensors(*cache, block)
    y = c.attn(q, i32([S - T]))
    check(y, cache, block, some_queries(1, T, H * rep), q, [S - T])
    assert status() == 0


# ---------------------------------------------------------------- many steps of the online softmax
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("B,T,Hq,H,D,S,dtype", [
    (1, 1, 8, 2, 128, 120000, "bf16"), (1, 1, 8, 2, 128, 120000, "fp32"), (1, 1, 8, 1, 64, 250000, "bf16"),
    (1, 1, 8, 1, 64, 250000, "fp32"), (1, 1, 8, 2, 256, 70000, "bf16"), (1, 1, 8, 2, 256, 70000, "fp32"),
    (2, 3, 8, 2, 128, 70000, "bf16"), (2, 3, 8, 2, 128, 70000, "fp32"), (1, 4, 16, 1, 64, 200000, "bf16"),
    (1, 4, 16, 1, 64, 200000, "fp32"), (1, 20, 8, 1, 256, 40000, "bf16"), (1, 30, 8, 2, 192, 40000, "fp32"),
    (1, 25, 8, 2, 128, 60000, "bf16"), (1, 25, 8, 2, 80, 60000, "bf16"), (1, 70, 8, 2, 128, 40000, "bf16"),
    (2, 130, 8, 2, 64, 20000, "bf16"), (2, 90, 16, 8, 128, 16384, "bf16")])
def test_long_runs(B, T, Hq, H, D, S, dtype, masked):
    """Scores that rise and fall by some 2^60 along the rows and value scales that double four times over and over: references and
    factors move in most steps, and each warp and CTA takes several. With masks over a third of the rows and sinks."""
    block = 16
    cache = rand_cache(S, B, H, S, D, block)
    wave = (torch.arange(S, device="cuda") % 3000 - 1500).abs() / 750 - 1
    cache[0].copy_((cache[0] * 0.3 + 85 * wave[:, None]).round())
    cache[3][:] *= 50 * sawtooth(cache[3].shape[2], 5, 1, 5)
    q = (rand_q(T, (B, T, Hq, D), dtype).float().abs() * (128 / D) ** 0.5).to(DT[dtype])
    mask = sinks = None
    if masked:
        g = torch.Generator(device="cuda").manual_seed(T)
        mask = torch.randn(B, T, S, device="cuda", generator=g)
        mask.masked_fill_(torch.rand(B, T, S, device="cuda", generator=g) < 0.3, -np.inf)
        sinks = torch.randn(Hq, device="cuda", generator=g)
    y = KVCache8.from_tensors(*cache, block).attn(q, i32([S - T] * B), mask=mask, sinks=sinks)
    check(y, cache, block, some_queries(B, T, Hq), q, [S - T] * B, mask, sinks)
    assert status() == 0


# ---------------------------------------------------------------- value scales far apart
@pytest.mark.parametrize("T,D", [(20, 128), (20, 64), (60, 128), (60, 64)])
@pytest.mark.parametrize("tiny", [1e-38, 1e-41, 1e-44])
def test_blocks_of_tiny_values_count_in_the_sum(T, D, tiny):
    """More than 64 bf16 queries a kv head: every other block holds values near fp32's smallest, and weighs in the
    softmax's sum like any other."""
    H, rep, S, block = 2, 4, 37900, 32
    cache = rand_cache(T + D, 1, H, S, D, block)
    cache[3][:, :, 1::2] = tiny
    q = rand_q(T, (1, T, H * rep, D), "bf16")
    c = KVCache8.from_tensors(*cache, block)
    y = c.attn(q, i32([S - T]))
    check(y, cache, block, some_queries(1, T, H * rep), q, [S - T])
    assert status() == 0


FAR = [(T, D, dtype) for T, dtype in ((1, "bf16"), (1, "fp32"), (5, "bf16"), (5, "fp32")) for D in (64, 128, 256)] + \
    [(T, D, "bf16") for T in (20, 60) for D in (64, 128)]


def hidden_case(T, D, dtype, r):
    """Blocks of values times r that a mask hides from all queries, the first of all among them."""
    H, rep, S, block = 2, 4, 120000 if T <= 5 else 38000, 32
    cache = rand_cache(T + D, 1, H, S, D, block)
    hide = torch.arange(cache[3].shape[2], device="cuda") * 7919 % 11 == 0
    cache[3][:, :, hide] *= r
    mask = torch.zeros(1, 1, S, device="cuda").masked_fill_(hide.repeat_interleave(block)[:S], -np.inf)
    q = rand_q(T, (1, T, H * rep, D), dtype)
    y = KVCache8.from_tensors(*cache, block).attn(q, i32([S - T]), mask=mask)
    check(y, cache, block, some_queries(1, T, H * rep), q, [S - T], mask)


def later_case(T, D, dtype, r):
    """The last token's values, in a block of their own, times r: the tokens before it do not see them."""
    H, rep, S, block = 2, 2 if T <= 5 else 4, 113, 16         # a tile of 10, 80 or 240 queries
    cache = rand_cache(T + D, 2, H, S, D, block)
    cache[3][:, :, -1] *= r
    q = rand_q(T, (2, T, H * rep, D), dtype)
    y = KVCache8.from_tensors(*cache, block).attn(q, i32([S - T, S - T]))
    check(y, cache, block, some_queries(2, T, H * rep, 12), q, [S - T, S - T])


def light_case(T, D, dtype, r):
    """Blocks of values times r at low scores: they weigh what e^x r makes of them, next to nothing or nearly all."""
    H, rep, S, block = 2, 4, 120000 if T <= 5 else 38000, 32
    cache = rand_cache(T + D, 1, H, S, D, block)
    light = torch.arange(cache[3].shape[2], device="cuda") * 7919 % 11 == 0
    cache[3][:, :, light] *= r
    cache[0][:, :, light.repeat_interleave(block)[:S]] = -127
    q = rand_q(T, (1, T, H * rep, D), dtype).abs()
    y = KVCache8.from_tensors(*cache, block).attn(q, i32([S - T]))
    check(y, cache, block, some_queries(1, T, H * rep), q, [S - T])


@pytest.mark.parametrize("r", [1e4, 1e8, 1e30])
@pytest.mark.parametrize("case", [hidden_case, later_case, light_case])
@pytest.mark.parametrize("T,D,dtype", FAR)
def test_value_scales_far_apart(T, D, dtype, case, r):
    if case is later_case and T == 1:
        pytest.skip("one token: none before it")
    case(T, D, dtype, r)
    assert status() == 0


# ---------------------------------------------------------------- more sequences and tiles than CTAs
@pytest.mark.parametrize("B,T,Hq,H,D,S,dtype,long", [
    (3000, 1, 8, 2, 64, 90, "bf16", 0), (700, 2, 16, 4, 128, 64, "fp32", 0), (150, 1, 8, 4, 256, 3000, "bf16", 70),
    (600, 1, 16, 2, 128, 5000, "fp32", 9), (1, 700, 4, 2, 256, 1500, "bf16", 0), (3, 300, 8, 2, 64, 900, "fp32", 0),
    (90, 20, 8, 2, 64, 1500, "bf16", 30), (40, 33, 16, 2, 128, 2500, "bf16", 11), (5, 500, 16, 4, 128, 700, "bf16", 0)])
def test_many_sequences_and_query_tiles(B, T, Hq, H, D, S, dtype, long):
    """More (sequence, query tile, head) segments than CTAs, of mixed lengths, some sequences without tokens: parts of a segment
    are joined where a border between two CTAs falls into it. Every `long`-th sequence is full, the others short."""
    block = 32
    cache = rand_cache(B, B, H, S, D, block)
    rng = np.random.default_rng(B + T)
    end = np.where(np.arange(B) % long == 0, S, rng.integers(T, T + 60, B)) if long else rng.integers(T, S + 1, B)
    cnt = np.where(rng.random(B) < (0.1 if B > 9 else 0), 0, T)
    cnt[[0, -1]] = T
    pos = end - T
    q = rand_q(B, (B, T, Hq, D), dtype)
    out = torch.full_like(q, 7)
    KVCache8.from_tensors(*cache, block).attn(q, i32(pos), i32(cnt), out=out)
    check(out, cache, block, [c for c in some_queries(B, T, Hq, 60) if cnt[c[0]]], q, pos)
    idle = torch.from_numpy(cnt == 0)
    assert (out[idle.cuda()] == 7).all() and torch.isfinite(out).all() and not (out[~idle.cuda()] == 7).all(-1).any()
    assert status() == 0


# ---------------------------------------------------------------- calls of several threads
FIRST_CALLS_AT_ONCE = """
import threading
import torch
from opennpu_b200 import libonpu as L
from opennpu_b200.kv8 import KVCache8
N = 16
L.load()
pos = torch.zeros(1, dtype=torch.int32, device="cuda")
x = torch.randn(1, 40, 12, 128, device="cuda").bfloat16()
torch.cuda.synchronize()
starts, caches, outs, errors = [threading.Barrier(N) for _ in range(3)], [None] * N, [None] * N, []
def work(i):
    try:
        with torch.cuda.stream(torch.cuda.Stream()):
            starts[0].wait()
            c = caches[i] = KVCache8(1, 2, 300, 128)
            starts[1].wait()
            c.append(x[:, :, 8:10], x[:, :, 10:], pos)
            starts[2].wait()
            outs[i] = c.attn(x[:, :40 if i % 2 else 1, :8], pos)
            torch.cuda.current_stream().synchronize()
    except Exception as e:
        errors.append(repr(e))
        [s.abort() for s in starts]
threads = [threading.Thread(target=work, args=(i,)) for i in range(N)]
[t.start() for t in threads]
[t.join() for t in threads]
assert not errors, errors
assert all(torch.equal(outs[i], outs[i % 2]) for i in range(N))
assert L.load().onpu_check_device() == 0
"""


def test_first_calls_of_several_threads_at_once():
    """In a fresh process: what the library looks up in a first call is there for the calls beside it."""
    import subprocess
    import sys

    from tests.conftest import ROOT
    for _ in range(3):
        r = subprocess.run([sys.executable, "-c", FIRST_CALLS_AT_ONCE], cwd=ROOT, capture_output=True, text=True, timeout=300)
        assert r.returncode == 0, r.stderr[-2000:]
