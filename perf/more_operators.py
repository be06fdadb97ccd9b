"""Timed cases of the paged KV cache in 4 bits: new keys and values written into
it with the position rotation (and the heads' norms) applied on the way
(paged_append_q4), tokens read back from it (paged_read_q4), and attention of a
chunk of new tokens, or of one, over it (paged_attention_q4).

A group is 32 neighbouring channels of a token's key or value in one head.  It
is held as codes c in 0..15, a zero point z in 0..15 and a scale s, a number
with four significant bits, and stands for (c - z) s, which 16 bits hold
exactly; see `_quantised`.  `run` computes a pass either in its plain form
(elementary torch operations, rounded once at the end) or, with own = True,
through torch.ops.tide.
"""
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
DEV = "cuda"


# ------------------------------------------------------------------ cases
def listed():
    return [
        # keys and values of a decode step of 256 requests, three quarters of
        # whose rows are still active, with the heads' norms
        dict(name="append_decode_256", op="append", dtype="bf16", tokens=256, live=0.75, hq=32,
             hkv=8, d=128, page=64, spare=500, norm=True, rotate=True, far=4000, mix=1),
        # those of one request, far into a long context: all latency
        dict(name="append_one_far", op="append", dtype="fp16", tokens=1, live=1.0, hq=32, hkv=8,
             d=128, page=16, spare=40, norm=False, rotate=True, far=130001, mix=2),
        # of the 16 x 2048 prefill of the 8B architecture
        dict(name="append_prefill_32768", op="append", dtype="bf16", tokens=32768, live=1.0, hq=32,
             hkv=8, d=128, page=64, spare=20, norm=False, rotate=True, far=0, mix=3),
        # GPT-2-small heads, positions in the embedding already
        dict(name="append_gpt2_d64", op="append", dtype="fp16", tokens=1999, live=1.0, hq=12,
             hkv=12, d=64, page=32, spare=7, norm=False, rotate=False, far=0, mix=4),
        # a few requests' tokens taken out of the cache
        dict(name="read_333", op="read", dtype="fp16", tokens=333, hole=0.1, hkv=12, d=64, page=16,
             spare=3, mix=5),
        # a whole long request taken out
        dict(name="read_26003", op="read", dtype="bf16", tokens=26003, hole=0.0, hkv=8, d=128,
             page=64, spare=9, mix=6),
        # one decode step of 256 sequences around 1024 positions, three
        # quarters of them still active after the checkpoints
        dict(name="attend_decode_256", op="attend", dtype="bf16", batch=256, new_lo=1, new_hi=1,
             ctx_lo=512, ctx_hi=1535, page=64, live=0.75, hq=32, hkv=8, d=128, mix=7),
        # single tokens of three requests with long contexts
        dict(name="attend_decode_long", op="attend", dtype="fp16", batch=3, new_lo=1, new_hi=1,
             ctx_lo=9001, ctx_hi=40001, page=16, live=1.0, hq=32, hkv=8, d=128, mix=8),
        # one token of two short requests: the smallest call
        dict(name="attend_decode_2", op="attend", dtype="bf16", batch=2, new_lo=1, new_hi=1,
             ctx_lo=3, ctx_hi=130, page=16, live=1.0, hq=14, hkv=2, d=128, mix=9),
        # a few drafted tokens of each request checked in one pass
        dict(name="attend_chunk_small", op="attend", dtype="bf16", batch=16, new_lo=1, new_hi=9,
             ctx_lo=0, ctx_hi=2100, page=32, live=1.0, hq=32, hkv=8, d=128, mix=10),
        # prompts of up to 512 tokens, GPT-2-small heads
        dict(name="attend_prompts_d64", op="attend", dtype="fp16", batch=8, new_lo=17, new_hi=512,
             ctx_lo=0, ctx_hi=0, page=64, live=1.0, hq=12, hkv=12, d=64, mix=11),
        # a 2048-token chunk of one long prompt
        dict(name="attend_chunk_long", op="attend", dtype="bf16", batch=1, new_lo=2048, new_hi=2048,
             ctx_lo=26003, ctx_hi=26003, page=128, live=1.0, hq=32, hkv=8, d=128, mix=12),
    ]


MOST_FLOPS = 9.1e11  # what the largest listed attention needs
MOST_SCORES = 2.2e9  # scores that the plain form holds at once


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    heads = [(32, 8, 128), (16, 2, 128), (8, 8, 128), (14, 2, 128), (12, 12, 64), (16, 4, 64),
             (6, 2, 64), (32, 1, 128)]
    while True:
        op = rng.choice(["append", "append", "read", "attend", "attend", "attend"])
        hq, hkv, d = rng.choice(heads)
        c = dict(op=op, dtype=rng.choice(["bf16", "fp16"]), hkv=hkv, d=d,
                 page=rng.choice([16, 32, 64, 128]), mix=rng.randrange(1, 1 << 20))
        if op == "attend":
            new = 1 if rng.random() < 0.5 else _log(rng, 2, 2048)
            ctx = _log(rng, 16, 40000)
            c.update(batch=_log(rng, 1, 256), new_lo=1 if new == 1 else rng.randint(0, new),
                     new_hi=new, ctx_lo=rng.randint(0, ctx), ctx_hi=ctx,
                     live=rng.choice([1.0, 0.5]), hq=hq)
        else:
            c.update(tokens=_log(rng, 1, 32768), spare=_log(rng, 1, 300))
        if op == "append":
            c.update(live=rng.choice([1.0, 0.6]), hq=hq, norm=rng.random() < 0.5,
                     rotate=rng.random() < 0.8, far=rng.choice([0, _log(rng, 1, 130000)]))
        if op == "read":
            c.update(hole=rng.choice([0.0, 0.1]))
        if op != "attend" or _fits(c):
            return c


def _fits(c):
    new, kv = _spans(c)
    scores = len(new) * c["hq"] * max(new) * max(kv)
    cells = len(new) * max(kv) * c["hkv"] * c["d"]
    held = sum(_spans(dict(c, live=1.0))[1]) * c["hkv"] * c["d"]
    return sum(new) and work(c)["flops"] <= MOST_FLOPS and scores <= MOST_SCORES \
        and cells <= 1 << 29 and held <= 1 << 29


def _lens(r, n, lo, hi):
    """n lengths of [lo, hi], both ends among them where there are two."""
    v = [r.randint(lo, hi) for _ in range(n)]
    v[0] = hi
    if n > 1:
        v[-1] = lo
    return v


def _alive(c, n):
    return max(1, int(n * c["live"]))


def _spans(c):
    """(new tokens, keys that the last of them sees) of each sequence that runs."""
    r = random.Random(c["mix"])
    new = _lens(r, c["batch"], c["new_lo"], c["new_hi"])
    ctx = _lens(r, c["batch"], c["ctx_lo"], c["ctx_hi"])
    n = _alive(c, c["batch"])
    return new[:n], [a + b for a, b in zip(ctx, new)][:n]


def work(c):
    held = c["hkv"] * c["d"] * 9.0 / 8  # bytes of a token's key and value in 4 bits
    if c["op"] == "attend":
        new, kv = _spans(c)
        seen = sum(q * (k - q) + q * (q + 1) / 2 for q, k in zip(new, kv))
        return {"bytes": 4.0 * c["d"] * c["hq"] * sum(new) + held * sum(kv),
                "flops": 4.0 * c["d"] * c["hq"] * seen}
    plain = 4.0 * c["hkv"] * c["d"]
    if c["op"] == "read":
        return {"bytes": c["tokens"] * (8 + held + plain), "flops": 0.0}
    # (what was written is read back, so that the pass has it as values)
    n = _alive(c, c["tokens"])
    return {"bytes": n * (16 + 4.0 * c["hq"] * c["d"] + 2 * plain + 2 * held), "flops": 0.0}


# ------------------------------------------------------------- the format
def _least(dtype):
    """The smallest scale of a group that is not all zeros."""
    return 2.0 ** -120 if dtype == torch.bfloat16 else 2.0 ** -21


def _quantised(x, dtype):
    """Codes, zero points and scales (fp32) of fp32 x [..., d].  With lo and hi
    the group's least and largest value, 0 among them: s is the smallest number
    of four significant bits of at least (hi - lo) / 15, z = round(-lo / s),
    c = round(x / s) + z within 0..15."""
    x = x.unflatten(-1, (-1, 32))
    lo, hi = x.amin(-1).clamp(max=0), x.amax(-1).clamp(min=0)
    t = (hi / 2 - lo / 2) / torch.full_like(hi, 7.5)
    s = ((t.view(torch.int32) + 0xFFFFF) & -0x100000).view(torch.float32)
    s = torch.where(t > 0, s.clamp(min=_least(dtype)), 0)
    by = torch.where(s > 0, s, 1)
    z = torch.round(-lo / by)
    c = (torch.round(x / by[..., None]) + z[..., None]).clamp(0, 15)
    return c.flatten(-2), z, s


def _bytes_of(c):
    """Bytes [..., d / 2] of codes [..., d]: eight channels are 32 bits, lowest
    first channels 0, 2, 4, 6, 1, 3, 5, 7."""
    c = c.to(torch.uint8).unflatten(-1, (-1, 8))[..., [0, 2, 4, 6, 1, 3, 5, 7]]
    return (c[..., ::2] | c[..., 1::2] << 4).flatten(-2)


def _codes_of(b):
    """fp32 codes [..., d / 32, 32] of bytes [..., d / 2]."""
    b = b.unflatten(-1, (-1, 4))
    c = torch.stack([b & 15, b >> 4], -1).flatten(-2)[..., [0, 4, 1, 5, 2, 6, 3, 7]]
    return c.flatten(-2).unflatten(-1, (-1, 32)).float()


def _packed(k, v, dtype):
    """Blocks [..., 18 d] of uint8 from fp32 k and v [..., 16, d]: the codes of
    the keys and of the values, a token after the other, then the keys' scales
    and the values' ([group, token % 4, token / 4], 16 bits each: the scale as
    a bf16, the zero point in its last four bits)."""
    codes, scales = [], []
    for x in (k, v):
        c, z, s = _quantised(x, dtype)
        codes.append(_bytes_of(c).flatten(-2))
        p = (s.view(torch.int32) >> 16 | z.int()).unflatten(-2, (4, 4))
        p = p.movedim(-1, -3).transpose(-1, -2).flatten(-3).to(torch.int16)
        scales.append(p.contiguous().view(torch.uint8))
    return torch.cat(codes + scales, -1)


def _value(c, z, s):
    """fp32 values of codes [..., d / 32, 32] (exact)."""
    return ((c - z[..., None]) * s[..., None]).flatten(-2)


def _opened(b):
    """Codes, zero points and scales (fp32) of keys and values [2, ..., 16, d]
    of blocks [..., 18 d]."""
    d = b.shape[-1] // 18
    c = torch.stack([b[..., :8 * d], b[..., 8 * d:16 * d]]).unflatten(-1, (16, -1))
    p = torch.stack([b[..., 16 * d:17 * d], b[..., 17 * d:]]).view(torch.int16).int()
    p = p.unflatten(-1, (-1, 4, 4)).transpose(-1, -2).movedim(-3, -1).flatten(-3, -2)
    s = ((p & 0xFFF0) << 16).view(torch.float32)
    return _codes_of(c), (p & 15).float(), s


# ----------------------------------------------------------------- inputs
def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _starts(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed * 7919 + c["mix"])
    return dict({"append": _prepare_append, "read": _prepare_read,
                 "attend": _prepare_attend}[c["op"]](c, g), op=c["op"], case=c)


def _keys(shape, g):
    """Keys: some channels are several times as large as the others."""
    x = torch.randn(shape, generator=g, device=DEV)
    return x * torch.exp(0.7 * torch.randn(shape[-1], generator=g, device=DEV))


def _filled(pages, c, g):
    """A cache of random keys and values, a slice of its pages at a time."""
    cache = torch.empty(pages, c["hkv"], c["page"] // 16, 18 * c["d"], dtype=torch.uint8,
                        device=DEV)
    dt = DTYPES[c["dtype"]]
    step = max(1, (1 << 26) // (c["hkv"] * c["page"] * c["d"]))
    for a in range(0, pages, step):
        n = min(step, pages - a)
        shape = (n, c["hkv"], c["page"] // 16, 16, c["d"])
        k, v = _keys(shape, g), torch.randn(shape, generator=g, device=DEV)
        cache[a:a + n] = _packed(k.to(dt).float(), v.to(dt).float(), dt)
    return cache


def _paged_slots(n, pages, page, g):
    """The slots of n tokens that fill pages of the pool one after the other."""
    at = torch.randperm(pages, generator=g, device=DEV)[:-(-n // page)]
    return (at[:, None] * page + torch.arange(page, device=DEV)).view(-1)[:n]


def _prepare_append(c, g):
    dt, d, hq, hkv, m = DTYPES[c["dtype"]], c["d"], c["hq"], c["hkv"], c["tokens"]
    n = _alive(c, m)
    pages = -(-m // c["page"]) + c["spare"]
    # q, k and v: column slices of one projection's output
    x = torch.cat([torch.randn(n, hq * d, generator=g, device=DEV), _keys((n, hkv * d), g),
                   torch.randn(n, hkv * d, generator=g, device=DEV)], 1).to(dt)
    if c["far"]:  # a token each of many requests
        slots = torch.randperm(pages * c["page"], generator=g, device=DEV)[:m]
    else:  # prompts: page after page
        slots = _paged_slots(m, pages, c["page"], g)
    rows = None
    if n < m:  # the rows that are still active, in order
        rows = torch.randperm(m, generator=g, device=DEV)[:n].sort()[0].to(torch.int32)
    freq = 1.0 / (500000.0 ** (torch.arange(0, d, 2, device=DEV).double() / d))
    w = [(1 + 0.2 * torch.randn(d, generator=g, device=DEV)).to(dt) for _ in range(2)]
    start = torch.randint(0, c["far"] + 1, (m,), generator=g, device=DEV)
    where = start if c["far"] else torch.arange(m, device=DEV) % 2048
    # the slots whose tokens this pass has written, which it reads back
    mine = slots if rows is None else slots[rows.long()]
    return dict(
        q=x[:, :hq * d].view(n, hq, d), k=x[:, hq * d:(hq + hkv) * d].view(n, hkv, d),
        v=x[:, (hq + hkv) * d:].view(n, hkv, d), slots=slots, rows=rows, mine=mine.contiguous(),
        positions=where, freq=freq.float() if c["rotate"] else None,
        qw=w[0] if c["norm"] else None, kw=w[1] if c["norm"] else None, eps=1e-6,
        cache=torch.zeros(pages, hkv, c["page"] // 16, 18 * d, dtype=torch.uint8, device=DEV),
        q_out=torch.empty(n, hq, d, dtype=dt, device=DEV),
        k_out=torch.zeros(n, hkv, d, dtype=dt, device=DEV),
        v_out=torch.zeros(n, hkv, d, dtype=dt, device=DEV))


def _prepare_read(c, g):
    dt, n = DTYPES[c["dtype"]], c["tokens"]
    pages = -(-n // c["page"]) + c["spare"]
    slots = _paged_slots(n, pages, c["page"], g)
    if c["hole"]:
        slots = torch.where(torch.rand(n, generator=g, device=DEV) < c["hole"], -1, slots)
    return dict(cache=_filled(pages, c, g), mine=slots.contiguous(),
                k_out=torch.zeros(n, c["hkv"], c["d"], dtype=dt, device=DEV),
                v_out=torch.zeros(n, c["hkv"], c["d"], dtype=dt, device=DEV))


def _tables_of(kv, page, g, spare):
    """A block table over randomly placed pages, what lies past a request's
    pages being -1, and the number of pages."""
    n = [-(-x // page) for x in kv]
    pages = sum(n) + spare
    place = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    at = torch.arange(max(max(n), 1), device=DEV)
    first = _i32(_starts(n)[:-1]).long()
    index = (first[:, None] + at).clamp_(max=pages - 1)
    return torch.where(at < _i32(n)[:, None], place[index], -1).contiguous(), pages


def _prepare_attend(c, g):
    new, kv = _spans(dict(c, live=1.0))
    n = _alive(c, c["batch"])
    dt = DTYPES[c["dtype"]]
    # the request of each sequence that runs: some of them, in any order
    order = torch.randperm(c["batch"], generator=g, device=DEV)
    where = torch.empty_like(order)
    where[order] = torch.arange(c["batch"], device=DEV)
    table, pages = _tables_of(kv, c["page"], g, 3)
    at = _starts(new[:n])
    q = torch.randn(at[-1], c["hq"], c["d"], generator=g, device=DEV).to(dt)
    return dict(q=q, cache=_filled(pages, c, g), table=table[where].contiguous(),
                lens=_i32(kv)[where], cu=_i32(at), single=c["new_lo"] == c["new_hi"] == 1,
                ids=order[:n].to(torch.int32), max_new=max(new[:n]), max_kv=max(kv),
                scale=c["d"] ** -0.5, out=torch.empty_like(q))


# -------------------------------------------------------------------- run
def run(s):
    if own:
        from tide_b200 import _native

        ops = _native.ops()
        if s["op"] == "attend":
            ops.paged_attention_q4(s["q"], s["cache"], s["table"], s["lens"],
                                   None if s["single"] else s["cu"], s["ids"], s["out"],
                                   s["max_kv"], s["scale"], None)
            return s["out"]
        if s["op"] == "append":
            ops.paged_append_q4(s["q"], s["k"], s["v"], s["slots"], s["rows"], None,
                                s["positions"], s["freq"], 1.0, s["qw"], s["kw"], s["eps"],
                                s["q_out"], s["cache"], None)
        ops.paged_read_q4(s["cache"], s["mine"], s["k_out"], s["v_out"], None)
        got = {"k": s["k_out"], "v": s["v_out"]}
        return dict(got, q=s["q_out"]) if s["op"] == "append" else got
    return {"append": _plain_append, "read": _plain_read, "attend": _plain_attend}[s["op"]](s)


# ------------------------------------------------------------ plain forms
def _turned(x, w, s):
    """x [n, heads, d] with the heads' norm and the rotation at the rows'
    positions, in 64 bits: angles of far positions, and keys next to the
    border between two codes."""
    x = x.double()
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"]) * w.double()
    if s["freq"] is None:
        return x
    at = s["positions"] if s["rows"] is None else s["positions"][s["rows"].long()]
    angle = (at.double()[:, None] * s["freq"].double())[:, None]
    a, b = x.chunk(2, -1)
    return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], -1)


def _plain_append(s):
    dt, d = s["k"].dtype, s["k"].shape[2]
    q = _turned(s["q"], s["qw"], s).to(dt)
    k = _turned(s["k"], s["kw"], s).float()
    cache, page = s["cache"], s["case"]["page"]
    place = (s["mine"] // page, s["mine"] % page // 16, s["mine"] % 16)
    for i, x in enumerate((k, s["v"].float())):
        c, z, sc = _quantised(x, dt)
        p = (sc.view(torch.int32) >> 16 | z.int()).to(torch.int16)
        codes = cache[..., 8 * d * i:8 * d * (i + 1)].unflatten(-1, (16, -1))
        codes[place[0], :, place[1], place[2]] = _bytes_of(c)
        scales = cache.view(torch.int16)[..., 8 * d + d // 2 * i:8 * d + d // 2 * (i + 1)]
        scales = scales.unflatten(-1, (-1, 4, 4))
        scales[place[0], :, place[1], :, place[2] % 4, place[2] // 4] = p
    return dict(_plain_read(s), q=q)


def _plain_read(s):
    cache, page, dt = s["cache"], s["case"]["page"], s["k_out"].dtype
    d = cache.shape[-1] // 18
    real = s["mine"] >= 0
    slot = s["mine"].clamp(min=0)
    pg, blk, tok = slot // page, slot % page // 16, slot % 16
    got = {}
    for i, name in enumerate(("k", "v")):
        c = cache[..., 8 * d * i:8 * d * (i + 1)].unflatten(-1, (16, -1))[pg, :, blk, tok]
        p = cache.view(torch.int16)[..., 8 * d + d // 2 * i:8 * d + d // 2 * (i + 1)]
        p = p.unflatten(-1, (-1, 4, 4))[pg, :, blk, :, tok % 4, tok // 4].int()
        x = _value(_codes_of(c), (p & 15).float(), ((p & 0xFFF0) << 16).view(torch.float32))
        got[name] = torch.where(real[:, None, None], x, 0).to(dt)
    return got


def _plain_attend(s):
    q, dt = s["q"], s["q"].dtype
    n, most = q.shape[0], s["max_new"]
    cu = s["cu"].long()
    # padded rows [B, most], and sequence and place of each of the n rows
    at = (cu[:-1, None] + torch.arange(most, device=DEV)).clamp_(max=n - 1)
    row = torch.arange(n, device=DEV)
    seq = torch.searchsorted(cu[1:].contiguous(), row, right=True)
    place = row - cu[seq]
    ids = s["ids"].long()
    B = ids.numel()
    kv = s["lens"][ids].long()
    wide = -(-s["max_kv"] // s["case"]["page"])
    pages = s["table"][ids].long().clamp(min=0)[:, :wide]
    # [2, B, pages, kv heads, blocks, 16, d] to [B, kv heads, keys, d]
    x = _value(*_opened(s["cache"][pages])).movedim(3, 2).flatten(3, 5)
    k, v = x[0], x[1]
    hkv = k.shape[1]
    G, d = q.shape[1] // hkv, q.shape[2]
    rows = q[at].float().view(B, most, hkv, G, d).permute(0, 2, 3, 1, 4)
    w = (rows.reshape(B, hkv, G * most, d) @ k.transpose(2, 3)).view(B, hkv, G, most, -1)
    w.mul_(s["scale"])
    last = (kv - (cu[1:] - cu[:-1]))[:, None] + torch.arange(most, device=DEV)
    hidden = torch.arange(w.shape[-1], device=DEV) > last[:, :, None]
    w.masked_fill_(hidden[:, None, None], float("-inf"))
    m = w.amax(-1, keepdim=True)
    w.sub_(m).exp_()
    o = w.view(B, hkv, G * most, -1) @ v
    o = o.view(B, hkv, G, most, d) / w.sum(-1, keepdim=True)
    return o.permute(0, 3, 1, 2, 4)[seq, place].reshape(n, -1, d).to(dt)


# ---------------------------------------------------------------- 64 bits
def exact(c, seed):
    s = prepare(c, seed)
    return {"append": _exact_append, "read": _exact_read, "attend": _exact_attend}[c["op"]](c, s)


def _exact_groups(x, dtype):
    """The values that groups of 64-bit x [..., d] are held as."""
    x = x.reshape(*x.shape[:-1], -1, 32)
    zero = torch.zeros((), dtype=torch.float64, device=DEV)
    lo, hi = torch.minimum(x.amin(-1), zero), torch.maximum(x.amax(-1), zero)
    t = (hi - lo) / 15
    mantissa, power = torch.frexp(t)  # 0.5 <= mantissa < 1
    s = torch.ldexp(torch.ceil(mantissa * 16) / 16, power)
    s = torch.where(t > 0, torch.clamp(s, min=_least(dtype)), torch.ones_like(s))
    z = torch.round(-lo / s)
    n = torch.round(x / s[..., None])
    n = torch.minimum(torch.maximum(n, -z[..., None]), 15 - z[..., None])
    return torch.where((t > 0)[..., None], n * s[..., None], 0).reshape(*x.shape[:-2], -1)


def _exact_append(c, s):
    dt, d = DTYPES[c["dtype"]], c["d"]
    at = s["positions"] if s["rows"] is None else s["positions"].index_select(0, s["rows"])
    got = {}
    for name, w in (("q", s["qw"]), ("k", s["kw"])):
        x = s[name].to(torch.float64)
        if w is not None:
            size = torch.linalg.vector_norm(x, dim=-1, keepdim=True)
            x = w.to(torch.float64) * x / torch.sqrt(size ** 2 / d + s["eps"])
        if s["freq"] is not None:
            # pairs (x_i, x_{i + d/2}) as complex numbers, turned by the angle
            turn = torch.outer(at.to(torch.float64), s["freq"].to(torch.float64))
            y = torch.complex(x[..., :d // 2], x[..., d // 2:])
            y = y * torch.polar(torch.ones_like(turn), turn)[:, None]
            x = torch.cat([y.real, y.imag], -1)
        got[name] = x
    # (a key is a 32-bit number before it is held in 4 bits)
    return {"k": _exact_groups(got["k"].float().double(), dt),
            "v": _exact_groups(s["v"].double(), dt), "q": got["q"]}


def _exact_token(cache, slot, page):
    """Keys and values [2, n, kv heads, d] in 64 bits of tokens at their slots,
    code by code."""
    d = cache.shape[-1] // 18
    b = cache[slot // page, :, slot % page // 16].long()  # the whole block of each
    t = (slot % 16)[:, None, None]
    out = []
    ch = torch.arange(d, device=DEV)
    nibble = torch.tensor([0, 4, 1, 5, 2, 6, 3, 7], device=DEV)[ch % 8]
    for i in range(2):
        byte = 8 * d * i + t * (d // 2) + ch // 8 * 4 + nibble // 2
        code = b.gather(-1, byte.expand(-1, b.shape[1], -1)) >> nibble % 2 * 4 & 15
        spot = 16 * d + d * i + 2 * (ch // 32 * 16 + t % 4 * 4 + t // 4)
        spot = spot.expand(-1, b.shape[1], -1)
        p = b.gather(-1, spot) | b.gather(-1, spot + 1) << 8
        scale = torch.where(p >> 4 > 0, (1 + (p >> 4 & 7) / 8.0).double() *
                            torch.exp2((p >> 7 & 255).double() - 127), 0)
        out.append((code - (p & 15)).double() * scale)
    return torch.stack(out)


def _exact_read(c, s):
    real = s["mine"] >= 0
    got = []
    for a in range(0, c["tokens"], 4096):
        got.append(_exact_token(s["cache"], s["mine"][a:a + 4096].clamp(min=0), c["page"]))
    got = torch.where(real[:, None, None], torch.cat(got, 1), 0)
    return {"k": got[0], "v": got[1]}


def _exact_attend(c, s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    at, lens, ids = s["cu"].tolist(), s["lens"].tolist(), s["ids"].tolist()
    G = c["hq"] // c["hkv"]
    for i, r in enumerate(ids):
        n, m = at[i + 1] - at[i], lens[r]
        pos = torch.arange(m, device=DEV)
        slot = s["table"][r].long()[pos // c["page"]] * c["page"] + pos % c["page"]
        kv = torch.cat([_exact_token(s["cache"], slot[a:a + 4096], c["page"])
                        for a in range(0, m, 4096)], 1) if m else None
        for h in range(c["hq"] if n else 0):
            kh, vh = kv[0, :, h // G], kv[1, :, h // G]
            for a in range(0, n, 1024):
                b = min(n, a + 1024)
                see = m - n + b
                logit = torch.mm(s["q"][at[i] + a:at[i] + b, h].double(), kh[:see].t()) * s["scale"]
                later = torch.ones(b - a, see, dtype=torch.bool, device=DEV).triu(m - n + a + 1)
                logit = logit.masked_fill(later, float("-inf"))
                out[at[i] + a:at[i] + b, h] = torch.softmax(logit, 1) @ vh[:see]
    return out
