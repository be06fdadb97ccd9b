"""Timed cases of the ragged serving operators: causal attention over packed
sequences of different lengths (packed_attention), attention of a chunk of new
tokens, or of one, over a paged cache (paged_attention), the write of new keys
and values into that cache (paged_append) and the page bookkeeping of a step
(page_tables).

`run` computes a pass either in its plain form (elementary torch operations in
32 bits, rounded once at the end) or, with own = True, through torch.ops.tide.
"""
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
DEV = "cuda"


# ------------------------------------------------------------------ cases
def listed():
    return [
        # survivors of a short live batch after the checkpoints: one to 48
        # tokens are left of each prompt, the call is all latency
        dict(name="packed_small_batch", op="packed", dtype="bf16", batch=6, lo=1, hi=48, keep=0.5,
             hq=32, hkv=8, d=128, fused=True, mix=1),
        # every token of the 16 x 2048 prefill of the 8B architecture
        dict(name="packed_prefill_16x2048", op="packed", dtype="bf16", batch=16, lo=2048, hi=2048,
             keep=1.0, hq=32, hkv=8, d=128, fused=True, mix=2),
        # the same prompts after checkpoints have let two fifths of the tokens
        # go: ragged survivors, zero keys in place of the others
        dict(name="packed_survivors_16", op="packed", dtype="bf16", batch=16, lo=301, hi=2047,
             keep=0.6, hq=32, hkv=8, d=128, fused=True, mix=3),
        # GPT-2-small heads, fp16, prompts of up to 512 tokens
        dict(name="packed_gpt2_d64", op="packed", dtype="fp16", batch=8, lo=17, hi=512, keep=1.0,
             hq=12, hkv=12, d=64, fused=True, mix=4),
        # one decode step of 256 sequences around 1024 positions, three
        # quarters of them still active after the checkpoints
        dict(name="paged_decode_256", op="paged", dtype="bf16", batch=256, new_lo=1, new_hi=1,
             ctx_lo=512, ctx_hi=1535, page=64, live=0.75, hq=32, hkv=8, d=128, mix=5),
        # single tokens of three requests with long contexts
        dict(name="paged_decode_long", op="paged", dtype="fp16", batch=3, new_lo=1, new_hi=1,
             ctx_lo=9001, ctx_hi=40001, page=16, live=1.0, hq=32, hkv=8, d=128, mix=6),
        # a few drafted tokens of each request checked in one pass
        dict(name="paged_chunk_small", op="paged", dtype="bf16", batch=16, new_lo=1, new_hi=9,
             ctx_lo=0, ctx_hi=2100, page=32, live=1.0, hq=32, hkv=8, d=128, mix=7),
        # a 2048-token chunk of one long prompt
        dict(name="paged_chunk_long", op="paged", dtype="bf16", batch=1, new_lo=2048, new_hi=2048,
             ctx_lo=26003, ctx_hi=26003, page=128, live=1.0, hq=32, hkv=8, d=128, mix=8),
        # the bookkeeping of a decode step: 256 requests, a few of them done
        dict(name="tables_decode_256", op="tables", batch=256, new_lo=1, new_hi=1, ctx_lo=1,
             ctx_hi=4000, done=0.05, page=64, width=128, short=False, mix=9),
        # a wave of new prompts, 64 requests of up to 2048 tokens
        dict(name="tables_prefill_64", op="tables", batch=64, new_lo=1, new_hi=2048, ctx_lo=0,
             ctx_hi=0, done=0.0, page=16, width=160, short=False, mix=10),
        # keys and values of a decode step
        dict(name="append_decode_256", op="append", dtype="bf16", rows=256, hkv=8, d=128, page=64,
             pages=512, hole=0.1, mix=11),
        # keys and values of a 16 x 2048 prefill
        dict(name="append_prefill_32768", op="append", dtype="bf16", rows=32768, hkv=8, d=128,
             page=16, pages=2300, hole=0.0, mix=12),
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
        op = rng.choice(["packed", "packed", "paged", "paged", "paged", "tables", "append"])
        mix = rng.randrange(1, 1 << 20)
        if op == "packed":
            hq, hkv, d = rng.choice(heads)
            hi = _log(rng, 1, 8192)
            c = dict(op=op, dtype=rng.choice(["bf16", "fp16"]), batch=_log(rng, 1, 64),
                     lo=rng.randint(0, hi), hi=hi, keep=rng.choice([1.0, 0.7, 0.3]), hq=hq,
                     hkv=hkv, d=d, fused=rng.random() < 0.7, mix=mix)
        elif op == "paged":
            hq, hkv, d = rng.choice(heads)
            new = 1 if rng.random() < 0.4 else _log(rng, 2, 2048)
            ctx = _log(rng, 16, 40000)
            c = dict(op=op, dtype=rng.choice(["bf16", "fp16"]), batch=_log(rng, 1, 256),
                     new_lo=1 if new == 1 else rng.randint(0, new), new_hi=new,
                     ctx_lo=rng.randint(0, ctx), ctx_hi=ctx, page=rng.choice([16, 32, 64, 128]),
                     live=rng.choice([1.0, 0.5]), hq=hq, hkv=hkv, d=d, mix=mix)
        elif op == "tables":
            hi = 1 if rng.random() < 0.4 else _log(rng, 2, 4096)
            page = rng.choice([16, 32, 64, 128])
            c = dict(op=op, batch=_log(rng, 1, 700), new_lo=rng.randint(0, hi), new_hi=hi,
                     ctx_lo=0, ctx_hi=_log(rng, 1, 8000), done=rng.choice([0.0, 0.1, 0.4]),
                     page=page, width=12200 // page, short=rng.random() < 0.2, mix=mix)
        else:
            page = rng.choice([16, 32, 64, 128])
            rows = _log(rng, 1, 32768)
            hkv, d = rng.choice([(8, 128), (2, 128), (1, 128), (12, 64), (3, 64)])
            c = dict(op=op, dtype=rng.choice(["bf16", "fp16"]), rows=rows, hkv=hkv, d=d, page=page,
                     pages=rows // page + _log(rng, 1, 256), hole=rng.choice([0.0, 0.1]), mix=mix)
        if _fits(c):
            return c


def _fits(c):
    if c["op"] in ("packed", "paged"):
        qn, kn = _spans(c)
        if not sum(qn):
            return False
        scores = len(qn) * c["hq"] * max(qn) * max(kn)
        cells = len(qn) * max(kn) * c["hkv"] * c["d"]
        return work(c)["flops"] <= MOST_FLOPS and scores <= MOST_SCORES and cells <= 1 << 29
    if c["op"] == "tables":
        new, _, _ = _requests(c)
        return 0 < sum(new) <= 131072
    return True


def _lens(r, n, lo, hi):
    """n lengths of [lo, hi], both ends among them where there are two."""
    v = [r.randint(lo, hi) for _ in range(n)]
    v[0] = hi
    if n > 1:
        v[-1] = lo
    return v


def _spans(c):
    """(new tokens, keys that the last of them sees) of each sequence that runs."""
    r = random.Random(c["mix"])
    if c["op"] == "packed":
        full = _lens(r, c["batch"], c["lo"], c["hi"])
        left = [n if c["keep"] == 1.0 else int(round(n * c["keep"])) for n in full]
        return left, left
    new = _lens(r, c["batch"], c["new_lo"], c["new_hi"])
    ctx = _lens(r, c["batch"], c["ctx_lo"], c["ctx_hi"])
    n = _alive(c)
    return new[:n], [a + b for a, b in zip(ctx, new)][:n]


def _alive(c):
    return max(1, int(c["batch"] * c["live"]))


def _requests(c):
    """(new tokens, tokens held, done) of each request."""
    r = random.Random(c["mix"])
    new = _lens(r, c["batch"], c["new_lo"], c["new_hi"])
    ctx = _lens(r, c["batch"], c["ctx_lo"], c["ctx_hi"])
    done = [r.random() < c["done"] and c["batch"] > 1 for _ in new]
    return [0 if d else n for n, d in zip(new, done)], ctx, done


def work(c):
    if c["op"] in ("packed", "paged"):
        qn, kn = _spans(c)
        seen = sum(q * (k - q) + q * (q + 1) / 2 for q, k in zip(qn, kn))
        return {"bytes": 2.0 * c["d"] * (2 * c["hq"] * sum(qn) + 2 * c["hkv"] * sum(kn)),
                "flops": 4.0 * c["d"] * c["hq"] * seen}
    if c["op"] == "tables":
        new, ctx, done = _requests(c)
        pages = sum(-(-(n + x) // c["page"]) for n, x in zip(new, ctx))
        return {"bytes": 12.0 * sum(new) + 16.0 * c["batch"] + 8.0 * pages, "flops": 0.0}
    return {"bytes": 2.0 * 4 * c["rows"] * c["hkv"] * c["d"] + 8.0 * c["rows"], "flops": 0.0}


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
    return dict({"packed": _prepare_packed, "paged": _prepare_paged, "tables": _prepare_tables,
                 "append": _prepare_append}[c["op"]](c, g), op=c["op"], case=c)


def _rows(c, n, g):
    """q, k and v of n tokens: column slices of one projection's output, or
    tensors of their own."""
    dt, d, hq, hkv = DTYPES[c["dtype"]], c["d"], c["hq"], c["hkv"]
    x = torch.randn(n, (hq + 2 * hkv) * d, generator=g, device=DEV).to(dt)
    q, k, v = x[:, :hq * d], x[:, hq * d:(hq + hkv) * d], x[:, (hq + hkv) * d:]
    if not c["fused"]:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    return q.view(n, hq, d), k.view(n, hkv, d), v.view(n, hkv, d)


def _prepare_packed(c, g):
    lens, _ = _spans(c)
    at = _starts(lens)
    q, k, v = _rows(c, at[-1], g)
    s = dict(q=q, k=k, v=v, cu=_i32(at), max_len=max(lens), scale=c["d"] ** -0.5, zeros=None,
             out=torch.empty(q.shape, dtype=q.dtype, device=DEV))
    if c["keep"] < 1.0:
        # a survivor's rank among the survivors and its position in the
        # prompt: the tokens between them have exited and hold zero keys
        gap = torch.rand(at[-1], generator=g, device=DEV) / c["keep"] * 2 * (1 - c["keep"])
        run_ = torch.cumsum(gap.double(), 0)
        first = torch.repeat_interleave(_i32(at[:-1]).long(), _i32(lens).long(), output_size=at[-1])
        s["zeros"] = (run_ - run_[first] + gap[first]).to(torch.int32)
    return s


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


def _prepare_paged(c, g):
    r = random.Random(c["mix"])
    new = _lens(r, c["batch"], c["new_lo"], c["new_hi"])
    ctx = _lens(r, c["batch"], c["ctx_lo"], c["ctx_hi"])
    kv = [a + b for a, b in zip(ctx, new)]
    n = _alive(c)
    dt = DTYPES[c["dtype"]]
    # the request of each sequence that runs: all of them in order, or those
    # that are still active
    order = torch.randperm(c["batch"], generator=g, device=DEV)
    where = torch.empty_like(order)
    where[order] = torch.arange(c["batch"], device=DEV)
    ids = order[:n].to(torch.int32)
    lens = _i32(kv)[where]  # request order[i] has the lengths of sequence i
    table, pages = _tables_of(kv, c["page"], g, 3)
    table = table[where].contiguous()
    shape = (pages, c["hkv"], c["page"], c["d"])
    at = _starts(new[:n])
    q = torch.randn(at[-1], c["hq"], c["d"], generator=g, device=DEV).to(dt)
    single = c["new_hi"] == 1 and c["new_lo"] == 1
    return dict(q=q, kc=torch.randn(shape, generator=g, device=DEV, dtype=dt),
                vc=torch.randn(shape, generator=g, device=DEV, dtype=dt), table=table, lens=lens,
                cu=_i32(at), single=single, ids=ids, max_new=max(new[:n]),
                max_kv=max(kv), scale=c["d"] ** -0.5, out=torch.empty_like(q))


def _prepare_tables(c, g):
    new, ctx, done = _requests(c)
    page, width = c["page"], c["width"]
    held = sum(-(-x // page) for x in ctx)
    need = sum(-(-(n + x) // page) for n, x in zip(new, ctx))
    table, pages = _tables_of(ctx, page, g, 1 + (need - held) // 2 if c["short"] else need + 5)
    wide = torch.full((c["batch"], width), -1, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table[:, :width]
    free = torch.full((pages,), -1, dtype=torch.int32, device=DEV)
    used = torch.zeros(pages, dtype=torch.bool, device=DEV)
    used[table[table >= 0].long()] = True
    left = (~used).nonzero()[:, 0].to(torch.int32)
    left = left[torch.randperm(left.numel(), generator=g, device=DEV)]
    free[:left.numel()] = left
    tokens = sum(new)
    return dict(ctx=_i32(ctx), new=_i32(new), done=_i32([int(x) for x in done]), free=free,
                n_free=_i32([pages - held]), table=wide, page=page, tokens=tokens,
                n_free_out=_i32([0]), kv=_i32([0] * c["batch"]), cu=_i32([0] * (c["batch"] + 1)),
                slots=torch.zeros(tokens + 8, dtype=torch.int64, device=DEV),
                pos=torch.zeros(tokens + 8, dtype=torch.int64, device=DEV))


def _prepare_append(c, g):
    n, dt, hkv, d = c["rows"], DTYPES[c["dtype"]], c["hkv"], c["d"]
    x = torch.randn(n, 2 * hkv * d, generator=g, device=DEV).to(dt)
    slots = torch.randperm(c["pages"] * c["page"], generator=g, device=DEV)[:n]
    if c["hole"]:
        out = torch.rand(n, generator=g, device=DEV) < c["hole"]
        out[0] = False
        slots = torch.where(out, -1, slots)
    shape = (c["pages"], hkv, c["page"], d)
    return dict(k=x[:, :hkv * d].view(n, hkv, d), v=x[:, hkv * d:].view(n, hkv, d), slots=slots,
                kc=torch.zeros(shape, dtype=dt, device=DEV),
                vc=torch.zeros(shape, dtype=dt, device=DEV), page=c["page"])


# -------------------------------------------------------------------- run
def run(s):
    if own:
        from tide_b200 import _native

        ops = _native.ops()
        if s["op"] == "packed":
            ops.packed_attention(s["q"], s["k"], s["v"], s["cu"], s["zeros"], s["out"], s["scale"],
                                 None)
            return s["out"]
        if s["op"] == "paged":
            ops.paged_attention(s["q"], s["kc"], s["vc"], s["table"], s["lens"],
                                None if s["single"] else s["cu"], s["ids"], s["out"], s["max_kv"],
                                s["scale"], None)
            return s["out"]
        if s["op"] == "tables":
            ops.page_tables(s["ctx"], s["new"], s["done"], s["free"], s["n_free"], s["table"],
                            s["page"], s["n_free_out"], s["kv"], s["cu"], s["slots"], s["pos"],
                            None)
            return _tables_out(s)
        ops.paged_append(s["k"], s["v"], s["slots"], None, None, s["kc"], s["vc"], None)
        return {"k": s["kc"], "v": s["vc"]}
    return {"packed": _plain_packed, "paged": _plain_paged, "tables": _plain_tables,
            "append": _plain_append}[s["op"]](s)


def _tables_out(s):
    return {"free": s["free"], "n_free": s["n_free_out"], "table": s["table"], "kv": s["kv"],
            "cu": s["cu"], "slots": s["slots"], "positions": s["pos"]}


# ------------------------------------------------------------ plain forms
def _plain_attention(q, k, v, last, zeros, scale):
    """softmax(scale q k^T) v of padded rows q [B, Sq, hq, d] over k and v
    [B, Sk, hkv, d] in 32 bits: a query sees keys 0..last [B, Sq], and `zeros`
    more (or None) whose key and value are zero."""
    B, Sq, hq, d = q.shape
    hkv = k.shape[2]
    G = hq // hkv
    rows = q.float().view(B, Sq, hkv, G, d).permute(0, 2, 3, 1, 4).reshape(B, hkv, G * Sq, d)
    s = (rows @ k.float().permute(0, 2, 3, 1)).view(B, hkv, G, Sq, -1)
    s.mul_(scale)
    hidden = torch.arange(k.shape[1], device=DEV) > last[:, :, None]
    s.masked_fill_(hidden[:, None, None], float("-inf"))
    m = s.amax(-1, keepdim=True)
    if zeros is not None:
        z = zeros.float()[:, None, None, :, None]
        m = torch.where(z > 0, m.clamp(min=0), m)
    m = torch.where(m == float("-inf"), 0, m)
    s.sub_(m).exp_()
    total = s.sum(-1, keepdim=True)
    if zeros is not None:
        total = total + z * torch.exp(-m)
    o = s.view(B, hkv, G * Sq, -1) @ v.float().permute(0, 2, 1, 3)
    o = o.view(B, hkv, G, Sq, d) / torch.where(total == 0, 1, total)
    return o.permute(0, 3, 1, 2, 4).reshape(B, Sq, hq, d)


def _padded(cu, n, most):
    """Row of each place of the padded layout [B, most] (kept inside the n
    rows), and sequence and place of each of the n rows."""
    cu = cu.long()
    at = (cu[:-1, None] + torch.arange(most, device=DEV)).clamp_(max=n - 1)
    row = torch.arange(n, device=DEV)
    seq = torch.searchsorted(cu[1:].contiguous(), row, right=True)
    return at, seq, row - cu[seq]


def _plain_packed(s):
    n, most = s["q"].shape[0], s["max_len"]
    at, seq, place = _padded(s["cu"], n, most)
    last = torch.arange(most, device=DEV).expand(at.shape)
    zeros = None if s["zeros"] is None else s["zeros"][at]
    o = _plain_attention(s["q"][at], s["k"][at], s["v"][at], last, zeros, s["scale"])
    return o[seq, place].to(s["q"].dtype)


def _plain_paged(s):
    n, most = s["q"].shape[0], s["max_new"]
    at, seq, place = _padded(s["cu"], n, most)
    ids = s["ids"].long()
    B = ids.numel()
    new = (s["cu"][1:] - s["cu"][:-1]).long()
    kv = s["lens"][ids].long()
    pages = s["table"][ids].long().clamp(min=0)
    _, hkv, page, d = s["kc"].shape
    wide = -(-s["max_kv"] // page)
    k = s["kc"][pages[:, :wide]].permute(0, 1, 3, 2, 4).reshape(B, -1, hkv, d)
    v = s["vc"][pages[:, :wide]].permute(0, 1, 3, 2, 4).reshape(B, -1, hkv, d)
    last = (kv - new)[:, None] + torch.arange(most, device=DEV)
    o = _plain_attention(s["q"][at], k, v, last, None, s["scale"])
    return o[seq, place].to(s["q"].dtype)


def _plain_tables(s):
    page, done = s["page"], s["done"] != 0
    free, table = s["free"].clone(), s["table"].clone()
    width = table.shape[1]
    col = torch.arange(width, device=DEV)
    # the pages of the requests that are done go back, in order
    back = torch.where(done, (s["ctx"].long() + page - 1) // page, 0)
    n1 = s["n_free"].long() + back.sum()
    spot = s["n_free"].long() + (back.cumsum(0) - back)[:, None] + col
    spot = torch.where(col < back[:, None], spot, free.numel())
    free = torch.cat([free, free[:1]]).scatter_(0, spot.view(-1), table.view(-1))[:-1]
    # and every other request gets what its new tokens need, from the top
    ctx = torch.where(done, 0, s["ctx"].long())
    new = s["new"].long()
    have = (ctx + page - 1) // page
    need = (ctx + new + page - 1) // page - have
    fits = have + need <= width
    need = torch.where(fits, need, 0)
    upto = need.cumsum(0)
    fits = fits & ((need == 0) | (upto <= n1))
    need = torch.where(fits, need, 0)
    taken = torch.where(need > 0, upto, 0).max()
    k = (upto - need)[:, None] + col - have[:, None]
    mine = (col >= have[:, None]) & (col < (have + need)[:, None])
    table = torch.where(mine, free[(n1 - 1 - k).clamp(0, free.numel() - 1)], table)
    cu = torch.cat([new.new_zeros(1), new.cumsum(0)])
    row = torch.arange(s["slots"].numel(), device=DEV)
    seq = torch.searchsorted(cu[1:].contiguous(), row, right=True).clamp_(max=ctx.numel() - 1)
    real = row < cu[-1]
    pos = torch.where(real, ctx[seq] + row - cu[seq], 0)
    slot = table[seq, (pos // page).clamp(max=width - 1)].long() * page + pos % page
    return {"free": free, "n_free": (n1 - taken).int(), "table": table,
            "kv": torch.where(fits, ctx + new, ctx).int(), "cu": cu.int(),
            "slots": torch.where(real & fits[seq], slot, -1), "positions": pos}


def _plain_append(s):
    page = s["page"]
    real = s["slots"] >= 0
    # a row without a slot writes what the first row with one writes
    src = torch.where(real, torch.arange(real.numel(), device=DEV), real.int().argmax())
    slot = s["slots"][src]
    s["kc"][slot // page, :, slot % page] = s["k"][src]
    s["vc"][slot // page, :, slot % page] = s["v"][src]
    return {"k": s["kc"], "v": s["vc"]}


# ---------------------------------------------------------------- 64 bits
def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "packed":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        at = s["cu"].tolist()
        for a, b in zip(at[:-1], at[1:]):
            z = None if s["zeros"] is None else s["zeros"][a:b].double()
            _exact_sequence(s["q"][a:b], s["k"][a:b], s["v"][a:b], z, s["scale"], out[a:b])
        return out
    if c["op"] == "paged":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        at = s["cu"].tolist()
        lens, ids = s["lens"].tolist(), s["ids"].tolist()
        for i, r in enumerate(ids):
            p = s["table"][r, :-(-lens[r] // c["page"])].long()
            k = s["kc"][p].transpose(1, 2).flatten(0, 1)[:lens[r]]
            v = s["vc"][p].transpose(1, 2).flatten(0, 1)[:lens[r]]
            _exact_sequence(s["q"][at[i]:at[i + 1]], k, v, None, s["scale"], out[at[i]:at[i + 1]])
        return out
    if c["op"] == "append":
        got = {}
        for name in ("k", "v"):
            flat = torch.zeros(c["pages"] * c["page"], c["hkv"], c["d"], dtype=torch.float64,
                               device=DEV)
            keep = (s["slots"] >= 0).nonzero()[:, 0]
            flat[s["slots"][keep]] = s[name][keep].double()
            got[name] = flat.view(c["pages"], c["page"], c["hkv"], c["d"]).transpose(1, 2)
        return got
    return None


def _exact_sequence(q, k, v, zeros, scale, out):
    """One sequence head by head: log-sum-exp weights in 64 bits, the queries
    being the last positions of the keys."""
    n, hq, _ = q.shape
    G = hq // k.shape[1]
    ahead = k.shape[0] - n
    for h in range(hq):
        kh, vh = k[:, h // G].double(), v[:, h // G].double()
        for a in range(0, n, 1024):
            b = min(n, a + 1024)
            see = ahead + b
            logit = torch.mm(q[a:b, h].double(), kh[:see].t()) * scale
            later = torch.ones(b - a, see, dtype=torch.bool, device=DEV).triu(ahead + a + 1)
            logit = logit.masked_fill(later, float("-inf"))
            norm = torch.logsumexp(logit, 1)
            if zeros is not None:
                norm = torch.logaddexp(norm, torch.log(zeros[a:b]))
            out[a:b, h] = torch.mm(torch.exp(logit - norm[:, None]), vh[:see])
