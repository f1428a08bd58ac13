"""Serving a batch of requests from a paged cache of keys and values in 8 bits, as it is measured.

Block tables and slot maps from request lengths, new keys and values into the cache (and back), attention over it for single
tokens, draft tokens and prompts, and the log probabilities of the tokens that were given, with entropy and alternatives.

The cache: blocks of `block` tokens, [blocks, kv heads, block, dim] codes of one byte (int8, or 4 exponent and 3 mantissa bits)
and one exponent byte per block and head: value = code * 2^(exponent - 127).

Where `own` is false `run` computes the operators with elementary torch operations; where it is true it calls nn_b200.
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
TOP = {"int8": 127.0, "e4m3": 448.0}
DTYPE = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # a step of eight conversations: the smallest call, all latency
        dict(name="tables 8 decode", kind="tables", requests=8, block=16, most=1, past=4000, mix=1),
        # a full server: some 300 requests, among them new prompts
        dict(name="tables 300 mixed", kind="tables", requests=300, block=32, most=700, past=9000, mix=2),
        # a decode step of 48 requests, one token each
        dict(name="append 48 decode int8", kind="append", fmt="int8", requests=48, most=1, past=3000, kv=8, dim=128, block=16, x="f32", mix=3),
        # prompts of about 4000 tokens each, bf16 rows
        dict(name="append prompts e4m3", kind="append", fmt="e4m3", requests=3, most=5000, past=100, kv=8, dim=128, block=32, x="bf16", mix=4),
        # one conversation of some 2000 tokens, the shape of the 8B decoder: latency
        dict(name="attend 1 x 2001 int8", kind="attend", fmt="int8", lengths=2001, requests=1, spread=0, rows=1, kv=8, group=4, dim=128, block=16, window=0, x="bf16", mix=5),
        # a decode step of 40 requests of very different lengths
        dict(name="attend 40 ragged e4m3", kind="attend", fmt="e4m3", lengths=12000, requests=40, spread=1, rows=1, kv=8, group=4, dim=128, block=32, window=0, x="bf16", mix=6),
        # two long documents, five query heads to a key head, f32 queries
        dict(name="attend 2 x 130001 int8", kind="attend", fmt="int8", lengths=130001, requests=2, spread=0, rows=1, kv=8, group=5, dim=128, block=64, window=0, x="f32", mix=7),
        # five draft tokens each to be checked, small heads, a sliding window
        dict(name="attend drafts int8", kind="attend", fmt="int8", lengths=3000, requests=11, spread=1, rows=5, kv=4, group=7, dim=64, block=16, window=1024, x="f32", mix=8),
        # a prompt's portion of 2000 tokens behind some 2000
        dict(name="attend prompt e4m3", kind="attend", fmt="e4m3", lengths=4100, requests=1, spread=0, rows=2000, kv=8, group=4, dim=128, block=16, window=0, x="bf16", mix=9),
        # the token that a step has chosen, with five alternatives
        dict(name="logprobs 1 row", kind="logprobs", rows=1, vocab=151936, top=5, x="f32"),
        # scoring a prompt's tokens
        dict(name="logprobs 129 rows", kind="logprobs", rows=129, vocab=151936, top=20, x="f32"),
        dict(name="logprobs 2000 rows", kind="logprobs", rows=2000, vocab=128259, top=1, x="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tables", "append", "append", "attend", "attend", "attend", "attend", "logprobs", "logprobs"])
    mix = rng.randrange(1 << 30)
    if kind == "tables":
        return dict(kind=kind, requests=_log_int(rng, 1, 1500), block=rng.choice([16, 32, 64, 128, 256]), most=rng.choice([1, 1, 5, 60]), past=_log_int(rng, 1, 20000), mix=mix)
    if kind == "append":
        fmt, kv, dim, block = rng.choice(["int8", "e4m3"]), rng.choice([1, 2, 4, 8, 16]), rng.choice([64, 128, 192, 256]), rng.choice([16, 32, 64, 128, 256])
        few = rng.random() < 0.5
        requests = _log_int(rng, 1, 300) if few else rng.randint(1, 3)
        return dict(kind=kind, fmt=fmt, requests=requests, most=rng.choice([1, 1, 4]) if few else _log_int(rng, 8, min(4000, 8000000 // (requests * kv * dim))),
                    past=_log_int(rng, 1, 4000), kv=kv, dim=dim, block=block, x=rng.choice(["bf16", "f32"]), mix=mix)
    if kind == "attend":
        form = rng.choice(["one", "one", "few", "prompt"])
        kv, group, dim = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16]), rng.choice([64, 128, 128, 192, 256])
        if form == "one":
            requests, rows = _log_int(rng, 1, 200), 1
            lengths = _log_int(rng, 1, min(130000, 250000000 // (requests * kv * dim)))
        elif form == "few":
            requests, rows = _log_int(rng, 1, 40), rng.randint(2, 9)
            lengths = _log_int(rng, rows, min(8000, 250000000 // (requests * kv * dim)))
        else:
            requests, rows = rng.randint(1, 2), _log_int(rng, 10, min(2000, 8000000 // (kv * group * dim)))
            lengths = rows + _log_int(rng, 1, min(4000, 22000000000 // (requests * rows * kv * group * dim)))
        return dict(kind=kind, fmt=rng.choice(["int8", "e4m3"]), lengths=lengths, requests=requests, spread=rng.choice([0, 1]), rows=rows, kv=kv, group=group, dim=dim,
                    block=rng.choice([16, 32, 64, 128, 256]), window=rng.choice([0, 0, _log_int(rng, 1, 4000)]), x=rng.choice(["bf16", "f32"]), mix=mix)
    vocab = _log_int(rng, 200, 152000)
    return dict(kind=kind, rows=_log_int(rng, 1, min(4000, 120000000 // vocab)), vocab=vocab, top=rng.choice([0, 1, 5, 20, 32]), x=rng.choice(["bf16", "f32"]))


# ------------------------------------------------------------------------------------------
# what a case says about its requests: host arithmetic from the case alone
# ------------------------------------------------------------------------------------------


def _requests(c):
    """(tokens held, tokens new) of every request."""
    r = random.Random(c["mix"])
    if c["kind"] == "attend":
        held, new = [], []
        for _ in range(c["requests"]):
            total = max(1, int(c["lengths"] * (r.random() ** 2 if c["spread"] else 1.0)))
            rows = min(total, c["rows"])
            held.append(total - rows)
            new.append(rows)
        return held, new
    held = [r.randint(0, c["past"]) for _ in range(c["requests"])]
    if c["most"] == 1:
        return held, [1] * c["requests"]
    if c["kind"] == "append":
        return held, [r.randint((c["most"] + 1) // 2, c["most"]) for _ in held]
    return held, [r.randint(1, c["most"]) if r.random() < 0.3 else (1 if r.random() < 0.9 else 0) for _ in held]


def _up(a, b):
    return -(-a // b)


def _seen(c):
    """Pairs of a row and a position it sees, and positions that some row of a request sees."""
    pairs = keys = 0
    for held, new in zip(*_requests(c)):
        first = None
        for i in range(new):
            p = held + i
            lo = max(0, p - c["window"] + 1) if c["window"] else 0
            first = lo if first is None else first
            pairs += p - lo + 1
        keys += held + new - first
    return pairs, keys


def work(c):
    if c["kind"] == "logprobs":
        n = c["rows"] * c["vocab"]
        return {"bytes": n * (4 if c["x"] == "f32" else 2) + c["rows"] * (12 + 8 * c["top"]), "flops": 6 * n}
    held, new = _requests(c)
    rows, reqs = sum(new), c["requests"]
    if c["kind"] == "tables":
        blocks = sum(_up(h + n, c["block"]) - _up(h, c["block"]) for h, n in zip(held, new))
        return {"bytes": 8 * reqs + 8 * blocks + 8 * reqs + 8 * rows, "flops": 4 * rows + 8 * reqs}
    width, es = c["kv"] * c["dim"], 4 if c["x"] == "f32" else 2
    if c["kind"] == "append":   # rows in, codes out, and the touched blocks back as bf16
        back = sum(h + n - h // c["block"] * c["block"] for h, n in zip(held, new))
        return {"bytes": 2 * rows * width * (es + 1) + 2 * back * width * 3, "flops": 2 * width * (3 * rows + back)}
    pairs, keys = _seen(c)
    return {"bytes": 2 * keys * width + 2 * rows * width * c["group"] * es, "flops": 4 * pairs * width * c["group"]}


# ------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _codes(g, fmt, shape):
    """Codes as a quantizer leaves them: most of the range used, values near zero the most frequent."""
    x = torch.randn(shape, device=DEV, generator=g, dtype=torch.bfloat16)
    if fmt == "int8":
        return (x * 30).round().clamp_(-127, 127).to(torch.int8).view(torch.uint8)
    return (x * 100).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)


def _i32(a):
    return torch.tensor(a, dtype=torch.int32, device=DEV)


def _pool(g, c, held, new):
    """Block tables over a pool of shuffled blocks: (table of all blocks, free blocks behind, blocks in all)."""
    need = [_up(h + n, c["block"]) for h, n in zip(held, new)]
    blocks = sum(need) + 3
    order = torch.randperm(blocks, device=DEV, generator=g).to(torch.int32)
    table = torch.full((len(need), max(need) + 1), -1, dtype=torch.int32, device=DEV)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = order[at:at + n]
        at += n
    return table, order[at:], blocks


def _sums(a):
    out = [0]
    for x in a:
        out.append(out[-1] + x)
    return out


def prepare(c, seed):
    g = _gen(seed)
    s = dict(case=c)
    if c["kind"] == "logprobs":
        x = torch.randn(c["rows"], c["vocab"], device=DEV, generator=g) * 2.5
        s["token"] = torch.randint(0, c["vocab"], (c["rows"],), device=DEV, generator=g, dtype=torch.int32)
        x[torch.arange(c["rows"], device=DEV), s["token"].long()] += 9.0   # what was given is mostly what the model expects
        s["logits"] = x.to(DTYPE[c["x"]])
        return s
    held, new = _requests(c)
    rows = sum(new)
    if c["kind"] == "tables":
        old = [_up(h, c["block"]) for h in held]
        need = [_up(h + n, c["block"]) for h, n in zip(held, new)]
        fresh = sum(need) - sum(old)
        order = torch.randperm(sum(need) + 3, device=DEV, generator=g).to(torch.int32)
        s["past"], s["count"], s["free"], s["rows"] = _i32(held), _i32(new), order[:fresh + 3].contiguous(), rows
        s["table"] = torch.full((len(held), max(need) + 1), -1, dtype=torch.int32, device=DEV)
        at = fresh + 3
        for r, n in enumerate(old):
            s["table"][r, :n] = order[at:at + n]
            at += n
        if own:
            from nn_b200 import kv_cache
            s["batch"] = kv_cache.KvBatch(len(held), s["table"].shape[1], rows, c["block"])
            s["batch"].table.copy_(s["table"])
        return s
    table, _, blocks = _pool(g, c, held, new)
    shape = (blocks, c["kv"], c["block"], c["dim"])
    s["k"], s["v"] = _codes(g, c["fmt"], shape), _codes(g, c["fmt"], shape)
    base = 122 if c["fmt"] == "int8" else 120   # values of about one
    s["k_exp"] = torch.randint(base - 1, base + 2, shape[:2], device=DEV, generator=g).to(torch.uint8)
    s["v_exp"] = torch.randint(base - 1, base + 2, shape[:2], device=DEV, generator=g).to(torch.uint8)
    s["table"], s["length"], s["row_start"] = table, _i32([h + n for h, n in zip(held, new)]), _i32(_sums(new))
    if c["kind"] == "append":
        spread = (torch.randn(c["kv"], c["dim"], device=DEV, generator=g) * 0.7).exp()   # some channels of the keys are larger
        s["xk"] = (torch.randn(rows, c["kv"], c["dim"], device=DEV, generator=g) * spread).to(DTYPE[c["x"]])
        s["xv"] = torch.randn(rows, c["kv"], c["dim"], device=DEV, generator=g).to(DTYPE[c["x"]])
        slots, touched = [], []
        for r, (h, n) in enumerate(zip(held, new)):
            p = torch.arange(h // c["block"] * c["block"], h + n, device=DEV)
            touched.append(table[r, p // c["block"]] * c["block"] + p % c["block"])
            slots.append(touched[-1][h - h // c["block"] * c["block"]:])
        s["slots"], s["touched"] = torch.cat(slots).to(torch.int32), torch.cat(touched).to(torch.int32)
    else:
        s["q"] = torch.randn(rows, c["kv"] * c["group"], c["dim"], device=DEV, generator=g).to(DTYPE[c["x"]])
    if own:
        from nn_b200 import kv_cache
        s["cache"] = kv_cache.KvCache(blocks, c["kv"], c["dim"], c["block"], kv_cache.INT8 if c["fmt"] == "int8" else kv_cache.E4M3)
        for name in ("k", "v", "k_exp", "v_exp"):
            getattr(s["cache"], name).copy_(s[name])
            del s[name]
        if c["kind"] == "attend":
            s["batch"] = kv_cache.KvBatch.from_tensors(table, s["length"], s["row_start"], c["block"])
    return s


# ------------------------------------------------------------------------------------------
# the plain forms
# ------------------------------------------------------------------------------------------


def _decode(fmt, codes):
    return codes.view(torch.int8 if fmt == "int8" else torch.float8_e4m3fn).float()


def _encode(fmt, x):
    """Codes of values already divided by their scale."""
    top = TOP[fmt]
    x = torch.where(x.isnan(), 0.0, x).clamp(-top, top)
    return x.round().to(torch.int8).view(torch.uint8) if fmt == "int8" else x.to(torch.float8_e4m3fn).view(torch.uint8)


def _power(e):
    """2^(e - 127) from its bits, 0 < e < 255 (below: zero)."""
    return (e.int().clamp_min(0) << 23).view(torch.float32)


def _exponent(fmt, amax):
    """Exponent byte of the least power of two under which `amax` does not pass the largest code."""
    m, e = torch.frexp(amax)                 # amax = m 2^e, m in [1/2, 1)
    top_m, top_e = (127.0 / 128.0, 7) if fmt == "int8" else (448.0 / 512.0, 9)
    e = e - top_e + (m > top_m).int()
    return torch.where(amax > 0, e + 127, 0).clamp(7, 253)


def _plain_tables(s):
    c = s["case"]
    B, past, count, free, table = c["block"], s["past"].long(), s["count"].long(), s["free"], s["table"].clone()
    total = past + count
    old, need = (past + B - 1) // B, (total + B - 1) // B
    fresh = need - old
    first = torch.cumsum(fresh, 0) - fresh
    col = torch.arange(table.shape[1], device=DEV)[None]
    new = (col >= old[:, None]) & (col < need[:, None])
    at = (first[:, None] + col - old[:, None]).clamp(0, free.numel() - 1)
    table = torch.where(new, free[at], table)
    ends = torch.cumsum(count, 0)
    start = torch.cat([torch.zeros(1, dtype=torch.long, device=DEV), ends])
    row = torch.arange(s["rows"], device=DEV)
    req = torch.searchsorted(ends, row, right=True)
    pos = past[req] + row - start[req]
    slot = table[req, pos // B].long() * B + pos % B
    i32 = torch.int32
    return dict(table=table, length=total.to(i32), row_start=start.to(i32), slot=slot.to(i32), position=pos.to(i32), used=fresh.sum().to(i32).reshape(1))


def _plain_append_one(fmt, codes, exps, x, slot, B):
    """One of keys and values: codes [blocks, kv, B, dim] and exponents [blocks, kv] in place."""
    slot = slot.long()
    blk, off = slot // B, slot % B
    uniq, inv = torch.unique(blk, return_inverse=True)
    x = x.float()
    amax = torch.where(x.isfinite(), x.abs(), 0.0).amax(2)
    top = torch.zeros(uniq.numel(), x.shape[1], device=DEV)
    top.scatter_reduce_(0, inv[:, None].expand(-1, x.shape[1]), amax, "amax")
    first = torch.full((uniq.numel(),), B, device=DEV).scatter_reduce_(0, inv, off, "amin")     # tokens that the block held before
    was = exps[uniq].int()
    now = torch.maximum(_exponent(fmt, top), torch.where(first[:, None] > 0, was, 0))
    held = torch.arange(B, device=DEV)[None, :] < first[:, None]
    again = _encode(fmt, _decode(fmt, codes[uniq]) * _power(127 + was - now)[:, :, None, None])
    codes[uniq] = torch.where(held[:, None, :, None], again, codes[uniq])
    exps[uniq] = now.to(torch.uint8)
    codes[blk, :, off] = _encode(fmt, x * _power(254 - now)[inv][:, :, None])


def _plain_read_one(fmt, codes, exps, slot, B):
    slot = slot.long()
    return (_decode(fmt, codes[slot // B, :, slot % B]) * _power(exps[slot // B])[:, :, None]).to(torch.bfloat16)


def _plain_attend(s):
    c = s["case"]
    B, kv, group, dim = c["block"], c["kv"], c["group"], c["dim"]
    held, new = _requests(c)
    y = torch.empty(s["q"].shape, dtype=torch.float32, device=DEV)
    at = 0
    for r, (h, n) in enumerate(zip(held, new)):
        total = h + n
        lo = max(0, h - c["window"] + 1) if c["window"] else 0
        pos = torch.arange(lo, total, device=DEV)
        blk, off = s["table"][r, pos // B].long(), pos % B
        k = _decode(c["fmt"], s["k"][blk, :, off]) * _power(s["k_exp"][blk])[:, :, None]
        v = _decode(c["fmt"], s["v"][blk, :, off]) * _power(s["v_exp"][blk])[:, :, None]
        q = s["q"][at:at + n].float().reshape(n, kv, group, dim).permute(1, 0, 2, 3).reshape(kv, n * group, dim)
        score = torch.matmul(q, k.permute(1, 2, 0)).reshape(kv, n, group, -1) * (1.0 / math.sqrt(dim))
        me = torch.arange(h, total, device=DEV)[:, None]
        see = pos[None] <= me
        if c["window"]:
            see &= me - pos[None] < c["window"]
        score = score.masked_fill(~see[None, :, None], -math.inf)
        p = (score - score.amax(-1, keepdim=True)).exp()
        p = (p / p.sum(-1, keepdim=True)).reshape(kv, n * group, -1)
        y[at:at + n] = torch.matmul(p, v.permute(1, 0, 2)).reshape(kv, n, group, dim).permute(1, 0, 2, 3).reshape(n, kv * group, dim)
        at += n
    return y.to(s["q"].dtype)


def _plain_logprobs(s):
    x, top = s["logits"].float(), s["case"]["top"]
    m = x.amax(1, keepdim=True)
    e = (x - m).exp()
    l = e.sum(1, keepdim=True)
    lse = m + l.log()
    out = dict(logprob=(x.gather(1, s["token"].long()[:, None]) - lse)[:, 0], entropy=(l.log() - (e * (x - m)).sum(1, keepdim=True) / l)[:, 0])
    if top:
        idx = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
        out.update(top_tokens=idx.to(torch.int32), top_logprobs=x.gather(1, idx) - lse)
    return out


def run(s):
    c = s["case"]
    if own:
        return _own(s)
    if c["kind"] == "tables":
        return _plain_tables(s)
    if c["kind"] == "append":
        for codes, exps, x in ((s["k"], s["k_exp"], s["xk"]), (s["v"], s["v_exp"], s["xv"])):
            _plain_append_one(c["fmt"], codes, exps, x, s["slots"], c["block"])
        return tuple(_plain_read_one(c["fmt"], codes, exps, s["touched"], c["block"]) for codes, exps in ((s["k"], s["k_exp"]), (s["v"], s["v_exp"])))
    if c["kind"] == "attend":
        return _plain_attend(s)
    return _plain_logprobs(s)


# ------------------------------------------------------------------------------------------
# the calls of a user
# ------------------------------------------------------------------------------------------


def _own(s):
    c = s["case"]
    if c["kind"] == "tables":
        b = s["batch"]
        b.build(s["past"], s["count"], s["free"])
        return dict(table=b.table, length=b.length, row_start=b.row_start, slot=b.slot, position=b.position, used=b.used)
    if c["kind"] == "append":
        s["cache"].append(s["xk"], s["xv"], s["slots"])
        return s["cache"].read(s["touched"], torch.bfloat16)
    if c["kind"] == "attend":
        return s["cache"].attend(s["q"], s["batch"], window=c["window"], max_rows=c["rows"])
    from nn_b200 import logprobs
    r = logprobs.token_logprobs(s["logits"], s["token"], c["top"])
    out = dict(logprob=r.logprob, entropy=r.entropy)
    if c["top"]:
        out.update(top_tokens=r.top_tokens, top_logprobs=r.top_logprobs)
    return out


# ------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------


def _two64(n):
    """2^n exactly."""
    return torch.tensor([2.0 ** i for i in range(-400, 401)], dtype=torch.float64, device=n.device)[n.long() + 400]


def _bits_e4m3(u):
    """The values of bytes of one sign, four exponent (bias 7) and three mantissa bits."""
    u = u.long()
    e, m = (u >> 3) & 15, (u & 7).double()
    mag = torch.where(e == 0, m * 2.0 ** -9, (1.0 + m / 8.0) * _two64(e - 7))
    return torch.where(u >= 128, -mag, mag)


def _values64(fmt, codes):
    u = codes.long()
    return torch.where(u >= 128, u - 256, u).double() if fmt == "int8" else _bits_e4m3(codes)


def _round64(fmt, x):
    """The nearest value that a code of the format stands for, ties to the even one."""
    if fmt == "int8":
        return x.round().clamp(-127, 127)
    step = _two64((x.abs().clamp_min(2.0 ** -6)).frexp().exponent - 4)
    return ((x / step).round() * step).clamp(-448, 448)


def _append64(c, codes, exps, x, slots, touched):
    """Block by block: values of the touched slots after the rows have come."""
    B, top = c["block"], TOP[c["fmt"]]
    x, out = x.double(), {}
    where = slots.tolist()
    runs, i = [], 0
    while i < len(where):
        j = i + 1
        while j < len(where) and where[j] == where[j - 1] + 1 and where[j] // B == where[i] // B:
            j += 1
        runs.append((i, j))
        i = j
    for i, j in runs:
        b, o = where[i] // B, where[i] % B
        amax = x[i:j].abs().amax((0, 2))
        e = torch.ceil(torch.log2(amax.clamp_min(1e-60) / top))
        e = torch.where(amax <= top * _two64(e - 1), e - 1, torch.where(amax > top * _two64(e), e + 1, e)).clamp_min(-120)
        old = exps[b].double() - 127
        if o:
            e = torch.maximum(e, old)
        block = torch.empty(c["kv"], o + j - i, c["dim"], dtype=torch.float64, device=DEV)
        scale = _two64(e)[:, None, None]
        if o:
            block[:, :o] = _round64(c["fmt"], _values64(c["fmt"], codes[b, :, :o]) * _two64(old)[:, None, None] / scale) * scale
        block[:, o:] = _round64(c["fmt"], x[i:j].permute(1, 0, 2) / scale) * scale
        out[b] = block
    t = touched.tolist()
    parts, i = [], 0
    while i < len(t):
        n = out[t[i] // B].shape[1]
        parts.append(out[t[i] // B].permute(1, 0, 2))
        i += n
    return torch.cat(parts)


def exact(c, seed):
    global own
    was, own = own, False
    try:
        s = prepare(c, seed)
    finally:
        own = was
    if c["kind"] == "tables":
        return None   # whole numbers
    if c["kind"] == "append":
        return (_append64(c, s["k"], s["k_exp"], s["xk"], s["slots"], s["touched"]), _append64(c, s["v"], s["v_exp"], s["xv"], s["slots"], s["touched"]))
    if c["kind"] == "logprobs":
        lp, en, tt, tl = [], [], [], []
        for x, t in zip(s["logits"], s["token"].tolist()):
            x = x.double()
            lse = torch.logsumexp(x, 0)
            lp.append(x[t] - lse)
            en.append(-((x - lse).exp() * (x - lse)).sum())
            if c["top"]:
                # the k-th largest value, everything above it, and of its equals the first ones
                kth = torch.topk(x, c["top"]).values[-1]
                idx = torch.cat([(x > kth).nonzero()[:, 0], (x == kth).nonzero()[:, 0]])[:c["top"]]
                idx = idx[torch.sort(-x[idx], stable=True).indices]
                tt.append(idx.to(torch.int32))
                tl.append(x[idx] - lse)
        out = dict(logprob=torch.stack(lp), entropy=torch.stack(en))
        if c["top"]:
            out.update(top_tokens=torch.stack(tt), top_logprobs=torch.stack(tl))
        return out
    if work(c)["flops"] > 4e11:
        return None
    B, out = c["block"], []
    start, length = s["row_start"].tolist(), s["length"].tolist()
    for r, total in enumerate(length):
        rows = range(start[r], start[r + 1])
        flat = (s["table"][r].long()[:, None] * B + torch.arange(B, device=DEV)[None]).reshape(-1)[:total]
        y = torch.empty(len(rows), c["kv"] * c["group"], c["dim"], dtype=torch.float64, device=DEV)
        for h in range(c["kv"]):
            k = _values64(c["fmt"], s["k"][flat // B, h, flat % B]) * _two64(s["k_exp"][flat // B, h].long() - 127)[:, None]
            v = _values64(c["fmt"], s["v"][flat // B, h, flat % B]) * _two64(s["v_exp"][flat // B, h].long() - 127)[:, None]
            for j in range(c["group"]):
                head = h * c["group"] + j
                sc = s["q"][rows.start:rows.stop, head].double() @ k.T / math.sqrt(c["dim"])
                away = torch.arange(total - len(rows), total, device=DEV)[:, None] - torch.arange(total, device=DEV)[None]
                sc[away < 0] = -math.inf
                if c["window"]:
                    sc[away >= c["window"]] = -math.inf
                y[:, head] = torch.softmax(sc, 1) @ v
        out.append(y)
    return torch.cat(out)
