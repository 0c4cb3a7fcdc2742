"""The 8-bit KV cache measured: rows quantised as they are written (and read back), rows read back,
and attention over the cache. Each case names the cache (B sequences of up to S rows, Hkv heads of D,
one scale per `block` rows and head) and the call (T tokens a sequence, of which cnt are valid, the
first at row pos). ``run`` computes it with plain torch operations, or through
``opennpu_b200.kv8`` where ``own`` is set."""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ---------------------------------------------------------------- cases
def _case(name, op, B, T, Hkv, D, S, block, dtype, rep=1, lo=None, hi=None, pad=False, sinks=False, mask=False):
    """lo, hi: the smallest and largest number of rows a sequence holds after the call."""
    hi = S if hi is None else hi
    return {"name": name, "op": op, "B": B, "T": T, "Hkv": Hkv, "rep": rep, "D": D, "S": S, "block": block,
            "dtype": dtype, "lo": hi if lo is None else lo, "hi": hi, "pad": pad, "sinks": sinks, "mask": mask}


def listed():
    return [
        # one decode token of one sequence written to a Qwen3-8B layer's cache: the smallest write
        _case("write one token", "append", 1, 1, 8, 128, 4096, 32, "bf16", hi=2745),
        # a decode step of a full batch, every sequence at its own length
        _case("write a batch's tokens", "append", 64, 1, 8, 128, 4096, 32, "bf16", lo=33, hi=4096),
        # four prompts of 2048 tokens appended behind an earlier turn that ended inside a block
        _case("write prompts", "append", 4, 2048, 8, 128, 4096, 32, "bf16", lo=2100, hi=2750),
        # a padded batch of short prompts, fp32 rows, an odd head size and small blocks
        _case("write padded fp32", "append", 3, 37, 4, 80, 256, 16, "fp32", lo=50, hi=90, pad=True),
        # whole sequences read back as bf16, for a prompt's own attention or to hand the cache on
        _case("read long", "read", 8, 8192, 8, 128, 8192, 32, "bf16"),
        # a few rows read back exactly, odd count, large heads
        _case("read odd fp32", "read", 2, 331, 2, 256, 700, 64, "fp32", lo=400, hi=650),
        # one decode token over 4096 rows of a Qwen3-8B layer, fp32 query as the decode step's other attention takes it
        _case("one token, 4k", "attn", 1, 1, 8, 128, 4096, 32, "fp32", rep=4),
        # a conversation's first tokens: a few dozen rows, heads of 64, sinks
        _case("one token, short", "attn", 1, 1, 8, 64, 128, 32, "fp32", rep=8, hi=77, sinks=True),
        # one decode token at a very long context, Qwen2.5-32B's heads
        _case("one token, 128k", "attn", 1, 1, 8, 128, 131072, 32, "bf16", rep=5, hi=131001),
        # a decode step of 64 sequences of mixed lengths, Qwen3-30B-A3B's heads
        _case("a batch's tokens", "attn", 64, 1, 4, 128, 8192, 32, "bf16", rep=8, lo=100, hi=8192),
        # five draft tokens a sequence checked at once, a mask over earlier rows and sinks
        _case("draft tokens", "attn", 8, 5, 8, 64, 4096, 32, "fp32", rep=8, lo=500, hi=4000, pad=True, sinks=True,
              mask=True),
        # 512 tokens of a prompt over 16k earlier rows, Qwen2.5-32B's heads
        _case("prompt chunk", "attn", 1, 512, 8, 128, 16896, 32, "bf16", rep=5, hi=16800),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Another case of the same ranges. Costs are capped by the largest listed ones."""
    caps = [work(c) for c in listed()]
    most = {k: max(c[k] for c in caps) for k in ("bytes", "flops")}
    while True:
        op = rng.choice(["append", "read", "attn", "attn", "attn"])
        dtype = rng.choice(["bf16", "fp32"])
        D = rng.choice([64, 80, 96, 112, 128, 128, 192, 256])
        Hkv, rep = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16])
        block, B = rng.choice([16, 32, 32, 64]), _log(rng, 1, 64)
        if op == "attn":
            kind = rng.choice(["one", "one", "draft", "chunk"])
            T = 1 if kind == "one" else rng.randint(2, 16) if kind == "draft" or dtype == "fp32" else _log(rng, 17, 512)
        else:
            T, rep = rng.choice([1, _log(rng, 2, 4096)]), 1
        hi = max(T, _log(rng, 1, 65536 if B == 1 else 16384))
        lo = rng.randint(min(T, hi), hi)
        S = hi + rng.randint(0, 200)
        if op == "read":
            lo = max(lo, T)
        c = _case("", op, B, T, Hkv, D, S, block, dtype, rep, lo, hi, pad=T > 1 and rng.random() < 0.4,
                  sinks=op == "attn" and rng.random() < 0.3, mask=op == "attn" and rng.random() < 0.3)
        del c["name"]
        w = work(c)
        plain = 4 * B * S * Hkv * D * 4 + 4 * B * Hkv * rep * T * S * 4      # the plain form's tensors
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"] and plain <= 24e9:
            return c


def _places(c):
    """(pos, cnt) of every sequence: rows held after the call spread over [lo, hi], padded batches with
    cnt from 1 to T."""
    B, T, span = c["B"], c["T"], c["hi"] - c["lo"] + 1
    pos, cnt = [], []
    for b in range(B):
        end = c["hi"] - (b * 7919) % span
        n = 1 + (b * 5 + 2) % T if c["pad"] else T
        cnt.append(min(n, end))
        pos.append(end - cnt[-1])
    return pos, cnt


def work(c):
    pos, cnt = _places(c)
    D, Hkv, blk, elt = c["D"], c["Hkv"], c["block"], 2 if c["dtype"] == "bf16" else 4
    if c["op"] == "attn":
        held = sum(p + n for p, n in zip(pos, cnt))
        scales = sum(-(-(p + n) // blk) for p, n in zip(pos, cnt))
        seen = sum(n * p + n * (n + 1) // 2 for p, n in zip(pos, cnt))
        Hq = Hkv * c["rep"]
        by = 2 * Hkv * (held * D + scales * 4) + 2 * sum(cnt) * Hq * D * elt
        by += 4 * Hq * c["sinks"] + 4 * c["mask"] * sum(n * (p + n) for p, n in zip(pos, cnt))
        return {"bytes": by, "flops": 4 * D * Hq * seen}
    back = sum(p % blk + n for p, n in zip(pos, cnt)) if c["op"] == "append" else sum(cnt)
    scales = sum((p + n - 1) // blk - p // blk + 1 for p, n in zip(pos, cnt))
    by = 2 * Hkv * (back * D * (1 + elt) + scales * 4)                      # read back
    fl = 2 * Hkv * D * back
    if c["op"] == "append":
        by += 2 * Hkv * (sum(cnt) * D * (elt + 1) + scales * 4)             # new rows in, codes out
        fl += 2 * Hkv * D * 3 * sum(cnt)
    return {"bytes": by, "flops": fl}


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    c = case
    B, T, Hkv, D, S, blk = c["B"], c["T"], c["Hkv"], c["D"], c["S"], c["block"]
    dev, dt = torch.device("cuda"), TYPES[c["dtype"]]
    g = torch.Generator(device=dev).manual_seed(seed)
    nb = -(-S // blk)

    def codes():
        r = torch.randn(B, Hkv, S, D, device=dev, dtype=torch.float16, generator=g)
        return r.mul_(36).round_().clamp_(-127, 127).to(torch.int8)

    def scales():
        return torch.rand(B, Hkv, nb, device=dev, generator=g) * 0.02 + 0.018

    st = {"case": c, "k": codes(), "v": codes(), "ks": scales(), "vs": scales()}
    pos, cnt = _places(c)
    st["pos"] = torch.tensor(pos, dtype=torch.int32, device=dev)
    st["cnt"] = torch.tensor(cnt, dtype=torch.int32, device=dev)
    if c["op"] == "append":
        # the projections' rows [K heads | V heads] of every token, as one GEMV writes them
        kv = torch.randn(B, T, 2 * Hkv, D, device=dev, generator=g).to(dt)
        st["new_k"], st["new_v"] = kv[:, :, :Hkv], kv[:, :, Hkv:]
        st["from"] = st["pos"] // blk * blk                                 # read back from the block's first row
        st["back"] = st["pos"] + st["cnt"] - st["from"]
        st["rows"] = max(p % blk + n for p, n in zip(pos, cnt))
    elif c["op"] == "read":
        st["from"], st["back"], st["rows"] = st["pos"], st["cnt"], T
    else:
        Hq = Hkv * c["rep"]
        st["q"] = torch.randn(B, T, Hq, D, device=dev, generator=g).to(dt)
        st["sinks"] = torch.randn(Hq, device=dev, generator=g) if c["sinks"] else None
        st["mask"] = None
        if c["mask"]:
            hide = torch.rand(B, T, S, device=dev, generator=g) < 0.1
            st["mask"] = torch.zeros(B, T, S, device=dev).masked_fill_(hide, float("-inf"))
    if own:
        from opennpu_b200 import kv8
        st["cache"] = kv8.KVCache8.from_tensors(st["k"], st["v"], st["ks"], st["vs"], blk)
    # rows of the outputs behind a sequence's cnt are left as they are: one buffer, zeros there
    if c["op"] == "attn":
        st["out"] = torch.zeros_like(st["q"])
    else:
        st["out"] = [torch.zeros(B, st["rows"], Hkv, D, device=dev, dtype=dt) for _ in range(2)]
    return st


# ---------------------------------------------------------------- one pass
def run(state):
    s, c = state, state["case"]
    if own:
        if c["op"] == "attn":
            return s["cache"].attn(s["q"], s["pos"], s["cnt"], mask=s["mask"], sinks=s["sinks"], out=s["out"])
        if c["op"] == "append":
            s["cache"].append(s["new_k"], s["new_v"], s["pos"], s["cnt"])
        k, v = s["cache"].read(s["from"], s["back"], out=s["out"])
        return {"k": k, "v": v, "ks": s["ks"], "vs": s["vs"]} if c["op"] == "append" else {"k": k, "v": v}
    if c["op"] == "attn":
        return _attn(s)
    if c["op"] == "append":
        _append(s, "k", "ks", s["new_k"])
        _append(s, "v", "vs", s["new_v"])
    k, v = _read(s, "k", "ks"), _read(s, "v", "vs")
    return {"k": k, "v": v, "ks": s["ks"], "vs": s["vs"]} if c["op"] == "append" else {"k": k, "v": v}


def _window(first, rows, S):
    """Rows first .. first + rows - 1 of every sequence, kept inside the cache: [B, rows] indices."""
    return (first.long()[:, None] + torch.arange(rows, device=first.device)).clamp(max=S - 1)


def _append(s, codes, scales, new):
    c, blk = s["case"], s["case"]["block"]
    B, T, Hkv, D, S = c["B"], c["T"], c["Hkv"], c["D"], c["S"]
    nw = (T + blk - 2) // blk + 1                                            # blocks a sequence can touch
    pos, cnt = s["pos"].long()[:, None], s["cnt"].long()[:, None]
    first = pos // blk
    row = first * blk + torch.arange(nw * blk, device=pos.device)            # [B, nw * blk]
    is_new, is_old = (row >= pos) & (row < pos + cnt), row < pos
    bi = torch.arange(B, device=pos.device)[:, None]
    x = new.float()[bi, (row - pos).clamp(0, T - 1)].transpose(1, 2)         # [B, Hkv, rows, D]
    x = torch.where(is_new[:, None, :, None], x, 0.0).view(B, Hkv, nw, blk, D)
    blocks = first + torch.arange(nw, device=pos.device)
    touched = is_new.view(B, nw, blk).any(-1)[:, None]                       # [B, 1, nw]
    kept = blocks.clamp(max=s[scales].shape[2] - 1)
    held = s[scales].gather(2, kept[:, None].expand(B, Hkv, nw))
    s_old = torch.where(is_old.view(B, nw, blk).any(-1)[:, None], held, 0.0)
    s_new = torch.maximum(s_old, (x.abs().amax((-1, -2)).double() / 127).float())
    wide = s_new.double()[..., None, None]                                   # the codes' borders need 64 bits
    q_new = torch.where(wide > 0, x.double() / wide, 0.0).round().clamp(-127, 127)
    at = row.clamp(max=S - 1)[:, None, :, None].expand(B, Hkv, nw * blk, D)
    old = s[codes].gather(2, at).view(B, Hkv, nw, blk, D).double()
    q_old = torch.where(wide > s_old.double()[..., None, None], old * s_old.double()[..., None, None] / wide, old).round()
    is_new, is_old = (m.view(B, 1, nw, blk, 1) for m in (is_new, is_old))
    q = torch.where(is_new, q_new, torch.where(is_old & touched[..., None, None], q_old, old)).to(torch.int8)
    inside = (row < S) & (row < pos + cnt)
    b, r = inside.nonzero(as_tuple=True)
    s[codes][b, :, row[b, r]] = q.view(B, Hkv, nw * blk, D)[b, :, r]
    b, w = touched[:, 0].nonzero(as_tuple=True)
    s[scales][b, :, blocks[b, w]] = s_new[b, :, w]


def _read(s, codes, scales):
    c, blk = s["case"], s["case"]["block"]
    at = _window(s["from"], s["rows"], c["S"])
    b = torch.arange(c["B"], device=at.device)[:, None]
    x = s[codes][b, :, at].float() * s[scales][b, :, at // blk][..., None]   # [B, rows, Hkv, D]
    valid = torch.arange(s["rows"], device=at.device) < s["back"][:, None]
    return torch.where(valid[..., None, None], x, 0.0).to(TYPES[c["dtype"]])


def _attn(s):
    c = s["case"]
    B, T, Hkv, D, S, blk, rep = c["B"], c["T"], c["Hkv"], c["D"], c["S"], c["block"], c["rep"]
    row = torch.arange(S, device=s["q"].device)
    K = s["k"].float() * s["ks"][:, :, row // blk, None]
    q = s["q"].float().view(B, T, Hkv, rep, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, T * rep, D)
    x = (torch.matmul(q, K.transpose(-1, -2)) * D ** -0.5).view(B, Hkv, T, rep, S)
    del K
    if s["mask"] is not None:
        x = x + s["mask"][:, None, :, None]
    i = torch.arange(T, device=row.device)
    seen = row[None, None] <= s["pos"][:, None, None] + i[None, :, None]     # [B, T, S]
    x = x.masked_fill_(~seen[:, None, :, None], float("-inf"))
    m = x.amax(-1, keepdim=True)
    if s["sinks"] is not None:
        sink = s["sinks"].view(1, Hkv, 1, rep, 1)
        m = torch.maximum(m, sink)
    m = torch.where(m == float("-inf"), 0.0, m)
    e = x.sub_(m).exp_()
    total = e.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + (sink - m).exp()
    V = s["v"].float() * s["vs"][:, :, row // blk, None]
    V = torch.where((row < (s["pos"] + s["cnt"])[:, None])[:, None, :, None], V, 0.0)
    y = torch.matmul(e.view(B, Hkv, T * rep, S), V).view(B, Hkv, T, rep, D)
    y = torch.where(total > 0, y / total, 0.0).permute(0, 2, 1, 3, 4).reshape(B, T, Hkv * rep, D)
    valid = i[None] < s["cnt"][:, None]
    return torch.where(valid[..., None, None], y, 0.0).to(TYPES[c["dtype"]])


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    c, s = case, prepare(case, seed)
    B, T, Hkv, D, blk, rep = c["B"], c["T"], c["Hkv"], c["D"], c["block"], c["rep"]
    pos, cnt = _places(c)
    f64 = torch.float64
    if c["op"] == "attn":
        out = torch.zeros(B, T, Hkv * rep, D, dtype=f64, device=s["q"].device)
        for b in range(B):
            n, p = cnt[b], pos[b]
            K, V = ((s[a][b, :, :p + n].to(f64) * s[z][b].to(f64).repeat_interleave(blk, 1)[:, :p + n, None])
                    for a, z in (("k", "ks"), ("v", "vs")))
            q = s["q"][b, :n].to(f64).unflatten(1, (Hkv, rep))
            x = torch.einsum("tgrd,gsd->gtrs", q, K) / math.sqrt(D)
            hidden = torch.ones(n, p + n, dtype=torch.bool, device=x.device).triu(p + 1)
            x = x.masked_fill(hidden[None, :, None], float("-inf"))
            if s["mask"] is not None:
                x = x + s["mask"][b, :n, :p + n].to(f64)[None, :, None]
            if s["sinks"] is not None:                                       # a column that has no value
                col = s["sinks"].to(f64).view(Hkv, 1, rep, 1).expand(Hkv, n, rep, 1)
                w = torch.softmax(torch.cat([x, col], -1), -1)[..., :-1]
            else:
                w = torch.softmax(x, -1)
            w = torch.nan_to_num(w, nan=0.0)                                 # a row with nothing left
            out[b, :n] = torch.einsum("gtrs,gsd->tgrd", w, V).flatten(1, 2)
        return out
    res = {}
    for codes, scales, new in (("k", "ks", "new_k"), ("v", "vs", "new_v")):
        q, sc = s[codes], s[scales]
        if c["op"] == "append":
            for b in range(B):
                p, end = pos[b], pos[b] + cnt[b]
                for i in range(p // blk, (end - 1) // blk + 1):
                    lo, hi = max(p, i * blk), min(end, (i + 1) * blk)
                    x = s[new][b, lo - p:hi - p].transpose(0, 1).to(f64)     # [Hkv, rows, D]
                    was = sc[b, :, i].clone() if lo > i * blk else torch.zeros_like(sc[b, :, i])
                    now = torch.maximum(was, (x.abs().amax((1, 2)) / 127).float())
                    grew = (was.to(f64) / now.to(f64)).nan_to_num(0.0)
                    if lo > i * blk:
                        held = q[b, :, i * blk:lo].to(f64) * was.to(f64)[:, None, None]
                        again = (held / now.to(f64)[:, None, None]).round().to(torch.int8)
                        q[b, :, i * blk:lo] = torch.where((grew < 1)[:, None, None], again, q[b, :, i * blk:lo])
                    y = (x / now.to(f64)[:, None, None]).nan_to_num(0.0).round().clamp(-127, 127)
                    q[b, :, lo:hi] = y.to(torch.int8)
                    sc[b, :, i] = now
        val = torch.zeros(B, s["rows"], Hkv, D, dtype=f64, device=q.device)
        start = [p // blk * blk if c["op"] == "append" else p for p in pos]
        for b in range(B):
            lo, hi = start[b], pos[b] + cnt[b]
            w = q[b, :, lo:hi].to(f64) * sc[b].to(f64).repeat_interleave(blk, 1)[:, lo:hi, None]
            val[b, :hi - lo] = w.transpose(0, 1)
        res[codes] = val
        if c["op"] == "append":
            res[scales] = sc.to(f64)
    return {"k": res["k"], "v": res["v"], "ks": res["ks"], "vs": res["vs"]} if c["op"] == "append" else res
