"""Plain 64-bit references of the ragged operators and the error bound that
their kernels are held to."""
from __future__ import annotations

import torch


def attention_rows(q, k, v, last, zeros, scale):
    """Rows q [n, hq, d] over keys k, v [m, hkv, d] in 64 bits: row i sees keys
    0..last[i] and zeros[i] more that are zero.  Returns the outputs and, for
    the error bound, sum_j w_j |v_j| and the largest sum_e |q_e k_e| * scale
    of a row."""
    n, hq, d = q.shape
    G = hq // k.shape[1]
    q, k, v = q.double(), k.double(), v.double()
    k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    see = torch.arange(k.shape[0], device=q.device)[None] <= last[:, None]  # [n, m]
    s = torch.einsum("nhd,mhd->hnm", q, k) * scale
    s = torch.where(see, s, float("-inf"))
    z = torch.zeros(n, dtype=torch.float64, device=q.device) if zeros is None else \
        zeros.clamp(min=0).double()
    top = s.amax(-1) if k.shape[0] else torch.full((hq, n), float("-inf"), device=q.device).double()
    top = torch.where(z > 0, top.clamp(min=0), top)
    top = torch.where(top.isinf() & (top < 0), 0.0, top)
    w = torch.exp(s - top[..., None])
    total = w.sum(-1) + z * torch.exp(-top)
    w = w / torch.where(total == 0, 1.0, total)[..., None]
    w = torch.where(see, w, 0.0)
    # a value row counts for the rows that see it only: 0 * NaN is no part of the sum
    o = torch.einsum("hnm,mhd->nhd", w, v.nan_to_num(0, 0, 0))
    size = torch.einsum("hnm,mhd->nhd", w, v.abs().nan_to_num(0, 0, 0))
    odd = torch.where(v.isfinite(), 0.0, v)
    if bool((odd != 0).any()):  # (a NaN is not 0 either)
        for j in odd.flatten(1).ne(0).any(1).nonzero()[:, 0].tolist():
            o = torch.where(see[:, j, None, None], o + odd[j], o)
    reach = (torch.einsum("nhd,mhd->hnm", q.abs(), k.abs()).nan_to_num(0, 0, 0) * see).amax(-1) \
        if k.shape[0] else torch.zeros_like(top)
    return o, size, (reach * scale).t()[..., None]


def attention_bound(ref, size, reach, n_keys, d, dtype):
    """What the kernels may be off: the output rounded once to `dtype`
    (eps / 2 of it), the weights rounded to `dtype` before they meet the values
    (eps / 2 of sum w |v|), scores summed in 32 bits (d products, each add
    within 2^-23 of the running size, so a weight is off by that much
    relatively, in the sum above and the one below), the exponential (2^-20)
    and the sums over the keys in 32 bits (2^-23 an add)."""
    eps = torch.finfo(dtype).eps
    tiny = torch.finfo(dtype).smallest_normal
    rel = eps / 2 + 2 * (d * 2.0 ** -23 * reach + 2.0 ** -20) + 2 * (n_keys + 2) * 2.0 ** -23
    return eps / 2 * ref.abs() + rel * size * (1 + eps) + tiny


def check_attention(got, ref, size, reach, n_keys, d, dtype):
    got = got.double()
    odd = ~ref.isfinite()
    assert torch.equal(got.isnan(), ref.isnan())
    assert torch.equal(got[odd & ~ref.isnan()], ref[odd & ~ref.isnan()])
    off = (got - ref).abs()[~odd]
    may = attention_bound(ref, size, reach, n_keys, d, dtype).expand(ref.shape)[~odd]
    assert bool((off <= may).all()), f"off by up to {(off / may).max().item():.3g} of the bound"


def packed_reference(q, k, v, lens, zeros, scale):
    outs = []
    a = 0
    for n in lens:
        z = None if zeros is None else zeros[a:a + n]
        last = torch.arange(n, device=q.device)
        outs.append(attention_rows(q[a:a + n], k[a:a + n], v[a:a + n], last, z, scale))
        a += n
    return [torch.cat(x) for x in zip(*outs)]


def gather_pages(cache, table_row, length):
    """Positions 0..length-1 of one request: [length, hkv, d]."""
    page = cache.shape[2]
    p = table_row[:-(-length // page)].long()
    return cache[p].transpose(1, 2).flatten(0, 1)[:length]


def paged_reference(q, kc, vc, tables, kv_lens, new, ids, scale):
    outs = []
    a = 0
    for n, r in zip(new, ids):
        L = kv_lens[r]
        k, v = gather_pages(kc, tables[r], L), gather_pages(vc, tables[r], L)
        last = torch.arange(n, device=q.device) + L - n
        outs.append(attention_rows(q[a:a + n], k, v, last, None, scale))
        a += n
    return [torch.cat(x) for x in zip(*outs)]


def page_tables_reference(ctx, new, done, free, n_free, tables, page, n_slots):
    """The step's bookkeeping with plain lists; free and tables are copied."""
    free, tables = list(free), [list(t) for t in tables]
    width = len(tables[0])
    avail = n_free
    ctx = list(ctx)
    for r in range(len(ctx)):
        if done and done[r]:
            for j in range(min(-(-ctx[r] // page), width)):
                free[avail] = tables[r][j]
                avail += 1
            ctx[r] = 0
    kv, cu, slots, pos, short = [], [0], [], [], False
    for r, n in enumerate(new):
        have, need = -(-ctx[r] // page), -(-(ctx[r] + n) // page) - -(-ctx[r] // page)
        if not n:
            need = 0
        ok = ctx[r] + n <= width * page
        if ok and need:
            short = short or need > avail
            ok = not short
        if ok:
            for j in range(need):
                avail -= 1
                tables[r][have + j] = free[avail]
        kv.append(ctx[r] + n if ok else ctx[r])
        cu.append(cu[-1] + n)
        for t in range(n):
            p = ctx[r] + t
            slots.append(tables[r][p // page] * page + p % page if ok else -1)
            pos.append(p)
    slots += [-1] * (n_slots - len(slots))
    pos += [0] * (n_slots - len(pos))
    return dict(free=free, n_free=avail, tables=tables, kv=kv, cu=cu, slots=slots, pos=pos)
