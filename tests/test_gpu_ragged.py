"""The ragged operators on the GPU against plain 64-bit references: attention
over packed sequences and over a paged cache, the paged append and the page
bookkeeping, at the lengths, head groups, masks and layouts where they can go
wrong.  The bound of each comparison is derived in ragged_helpers."""
import random

import pytest
import torch

from tests.ragged_helpers import (check_attention, gather_pages, packed_reference,
                                  page_tables_reference, paged_reference)
from tide_b200 import _native

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def starts(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


def rows(n, hq, hkv, d, dtype, seed, fused=True, size=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = (torch.randn(n, (hq + 2 * hkv) * d, generator=g, device=DEV) * size).to(dtype)
    q, k, v = x[:, :hq * d], x[:, hq * d:(hq + hkv) * d], x[:, (hq + hkv) * d:]
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    return q.view(n, hq, d), k.view(n, hkv, d), v.view(n, hkv, d)


def run_packed(q, k, v, lens, zeros=None, scale=None, out=None, err=None):
    out = torch.empty(q.shape, dtype=q.dtype, device=DEV) if out is None else out
    _native.ops().packed_attention(q, k, v, i32(starts(lens)), zeros, out,
                                   scale or q.shape[2] ** -0.5, err)
    return out


LENS = [[1], [0, 1, 2, 127, 128, 129, 0, 300], [64] * 5, [1000], [5, 0, 0, 777, 31]]


@pytest.mark.parametrize("lens", LENS, ids=str)
@pytest.mark.parametrize("hq,hkv,d,dtype,fused", [
    (8, 2, 128, torch.bfloat16, True), (4, 4, 64, torch.float16, True),
    (14, 2, 128, torch.float16, False), (6, 2, 64, torch.bfloat16, False),
    (16, 1, 128, torch.bfloat16, True)])
def test_packed_attention(lens, hq, hkv, d, dtype, fused):
    q, k, v = rows(sum(lens), hq, hkv, d, dtype, sum(lens) + hq, fused)
    out = run_packed(q, k, v, lens)
    ref = packed_reference(q, k, v, lens, None, d ** -0.5)
    check_attention(out, *ref, max(lens), d, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", [0.01, 6.0])
def test_packed_attention_flat_and_peaked_scores(dtype, size):
    """Scores from all alike to a few hundred apart, the largest ones late in
    the sequence, so that the running maximum moves again and again."""
    lens, hq, hkv, d = [700, 260], 4, 2, 128
    q, k, v = rows(sum(lens), hq, hkv, d, dtype, 5, False, size)
    k = (k * torch.linspace(0.2, 1.0, k.shape[0], device=DEV)[:, None, None].to(dtype)).contiguous()
    out = run_packed(q, k, v, lens)
    check_attention(out, *packed_reference(q, k, v, lens, None, d ** -0.5), max(lens), d, dtype)


@pytest.mark.parametrize("hq,hkv,d,dtype", [(8, 2, 128, torch.bfloat16), (3, 3, 64, torch.float16)])
def test_packed_attention_zero_keys(hq, hkv, d, dtype):
    """Zero keys as a count: against the reference's count, and against the
    same keys written out as zero rows (a live prefill's exited tokens)."""
    lens = [150, 1, 0, 260]
    n = sum(lens)
    q, k, v = rows(n, hq, hkv, d, dtype, 3, True, 2.0)
    zeros = torch.randint(-3, 400, (n,), generator=torch.Generator(device=DEV).manual_seed(1),
                          device=DEV, dtype=torch.int32)
    zeros[::5] = 0
    out = run_packed(q, k, v, lens, zeros)
    check_attention(out, *packed_reference(q, k, v, lens, zeros, d ** -0.5), 660, d, dtype)


def test_packed_attention_zero_keys_are_exited_tokens():
    """Survivors with their zero counts against the whole sequence with the
    exited tokens' keys and values zeroed."""
    S, hq, hkv, d, dtype = 333, 8, 2, 128, torch.bfloat16
    q, k, v = rows(S, hq, hkv, d, dtype, 8, False)
    keep = torch.rand(S, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV) < 0.6
    pos = keep.nonzero()[:, 0]
    zeros = (pos - torch.arange(pos.numel(), device=DEV)).to(torch.int32)
    out = run_packed(q[pos].contiguous(), k[pos].contiguous(), v[pos].contiguous(), [pos.numel()], zeros)
    kz, vz = k * keep[:, None, None], v * keep[:, None, None]
    ref = [x[pos] for x in packed_reference(q, kz, vz, [S], None, d ** -0.5)]
    check_attention(out, *ref, S, d, dtype)


@pytest.mark.parametrize("d", [64, 128])
def test_packed_attention_values_that_are_not_finite(d):
    """A NaN or infinity in a value (or key) row reaches the rows that see it
    and no others: not the earlier rows of its sequence, not the neighbours."""
    lens, hq, hkv, dtype = [100, 37, 300, 20], 4, 2, torch.bfloat16
    q, k, v = rows(sum(lens), hq, hkv, d, dtype, 9, False)
    at = starts(lens)
    v[at[1] + 5, 0, 3] = float("nan")
    v[at[2] + 200, 1, 7] = float("inf")
    v[at[2] + 201, 1, 8] = float("-inf")
    v[at[2] + 299] = float("nan")
    out = run_packed(q, k, v, lens)
    check_attention(out, *packed_reference(q, k, v, lens, None, d ** -0.5), max(lens), d, dtype)
    assert bool(out[at[3]:].isfinite().all()) and bool(out[:at[1] + 5].isfinite().all())
    k[at[2] + 150] = float("nan")
    out = run_packed(q, k, v, lens)
    assert bool(out[at[2]:at[2] + 150].isfinite().all()) and bool(out[at[3]:].isfinite().all())
    assert bool(out[at[2] + 150:at[3]].isnan().all())


def test_packed_attention_leaves_the_rows_behind_and_skips_bad_sequences():
    hq, hkv, d, dtype = 4, 1, 128, torch.float16
    q, k, v = rows(200, hq, hkv, d, dtype, 4)
    k[150:], v[150:] = float("nan"), float("nan")
    out = torch.full_like(q, 7.0)
    err = i32([0])
    run_packed(q, k, v, [40, 110], None, None, out, err)
    assert int(err) == 0 and bool((out[150:] == 7).all())
    ref = packed_reference(q[:150], k[:150], v[:150], [40, 110], None, d ** -0.5)
    check_attention(out[:150], *ref, 110, d, dtype)
    # a sequence past the rows, and one that ends before it starts
    for cu, fine in (([0, 40, 201], slice(0, 40)), ([40, 30, 90], slice(30, 90))):
        out.fill_(7.0)
        err.zero_()
        _native.ops().packed_attention(q, k, v, i32(cu), None, out, d ** -0.5, err)
        torch.cuda.synchronize()
        assert int(err) & 1
        assert bool((out[fine] != 7).any(-1).all())
        rest = torch.ones(200, dtype=torch.bool, device=DEV)
        rest[fine] = False
        assert bool((out[rest] == 7).all())


# ------------------------------------------------------------------ paged
def paged_case(new, ctx, hq, hkv, d, dtype, page, seed, n_req=None, junk=float("nan")):
    """Caches whose unused places hold `junk`, tables whose unused entries are
    far outside, requests in an order of their own."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    n_req = n_req or len(new)
    ids = torch.randperm(n_req, generator=torch.Generator().manual_seed(seed))[:len(new)].tolist()
    lens = [0] * n_req
    for i, r in enumerate(ids):
        lens[r] = ctx[i] + new[i]
    pages = [-(-n // page) for n in lens]
    total = sum(pages) + 2
    place = torch.randperm(total, generator=torch.Generator().manual_seed(seed + 1)).tolist()
    width = max(pages) + 1
    tables = [[place.pop() for _ in range(n)] + [1 << 30] * (width - n) for n in pages]
    kc = torch.full((total, hkv, page, d), junk, dtype=dtype, device=DEV)
    vc = kc.clone()
    for r, n in enumerate(lens):
        for j in range(0, n, page):
            m = min(page, n - j)
            for c in (kc, vc):
                c[tables[r][j // page], :, :m] = torch.randn(hkv, m, d, generator=g, device=DEV).to(dtype)
    q = torch.randn(sum(new), hq, d, generator=g, device=DEV).to(dtype)
    return q, kc, vc, i32(tables), lens, ids


def run_paged(q, kc, vc, tables, lens, new, ids, out=None, err=None, live=None, max_kv=None, single=False):
    out = torch.empty(q.shape, dtype=q.dtype, device=DEV) if out is None else out
    _native.ops().paged_attention(q, kc, vc, tables, i32(lens), None if single else i32(starts(new)),
                                  None if ids is None else i32(ids), out,
                                  max(lens) if max_kv is None else max_kv, q.shape[2] ** -0.5, err, live)
    return out


@pytest.mark.parametrize("new,ctx", [
    ([1], [0]), ([1, 5, 0, 64, 130], [0, 127, 40, 128, 1000]), ([200], [3000]), ([3, 2], [9000, 17]),
    ([33, 1, 300, 7], [0, 0, 0, 255])], ids=str)
@pytest.mark.parametrize("hq,hkv,d,dtype,page", [
    (8, 2, 128, torch.bfloat16, 16), (4, 4, 64, torch.float16, 64), (14, 2, 128, torch.float16, 128),
    (6, 2, 64, torch.bfloat16, 256), (32, 1, 128, torch.bfloat16, 32)])
def test_paged_attention_chunks(new, ctx, hq, hkv, d, dtype, page):
    q, kc, vc, tables, lens, ids = paged_case(new, ctx, hq, hkv, d, dtype, page, sum(new) + page, len(new) + 2)
    err = i32([0])
    out = run_paged(q, kc, vc, tables, lens, new, ids, err=err)
    check_attention(out, *paged_reference(q, kc, vc, tables, lens, new, ids, d ** -0.5), max(lens), d, dtype)
    assert int(err) == 0


@pytest.mark.parametrize("hq,hkv,d,dtype,page", [
    (8, 2, 128, torch.bfloat16, 16), (2, 2, 64, torch.float16, 64), (14, 2, 128, torch.float16, 128),
    (4, 2, 64, torch.bfloat16, 32), (32, 1, 128, torch.bfloat16, 32), (16, 2, 64, torch.float16, 256)])
@pytest.mark.parametrize("ctx", [[0], [0, 15, 16, 127, 128, 129, 1000, 2047], [30000, 5], [511] * 40],
                         ids=lambda c: f"{len(c)}x{c[0]}")
def test_paged_attention_single_tokens(hq, hkv, d, dtype, page, ctx):
    new = [1] * len(ctx)
    q, kc, vc, tables, lens, ids = paged_case(new, ctx, hq, hkv, d, dtype, page, len(ctx) + page, len(ctx) + 1)
    err = i32([0])
    out = run_paged(q, kc, vc, tables, lens, new, ids, err=err, single=True)
    ref = paged_reference(q, kc, vc, tables, lens, new, ids, d ** -0.5)
    check_attention(out, *ref, max(lens), d, dtype)
    assert int(err) == 0
    # the same with a bound far above the lengths (another split of the keys)
    wide = torch.cat([tables, tables[:, :1].expand(-1, 70000 // page)], 1).contiguous()
    out = run_paged(q, kc, vc, wide, lens, new, ids, max_kv=65536, single=True)
    check_attention(out, *ref, max(lens), d, dtype)


@pytest.mark.parametrize("single", [False, True])
def test_paged_attention_live_count_and_requests(single):
    """Sequences at or past the live count, requests that do not exist and
    lengths past the bound leave their rows as they were."""
    new = [1] * 6 if single else [1, 20, 3, 40, 5, 6]
    ctx = [100, 30, 7, 260, 4, 90]
    q, kc, vc, tables, lens, ids = paged_case(new, ctx, 8, 2, 128, torch.bfloat16, 32, 11)
    ref = paged_reference(q, kc, vc, tables, lens, new, ids, 128 ** -0.5)
    at = starts(new)
    for n in (0, 4, 6):
        out = torch.full_like(q, 7.0)
        run_paged(q, kc, vc, tables, lens, new, ids, out, live=i32([n]), single=single)
        check_attention(out[:at[n]], *[x[:at[n]] for x in ref], max(lens), 128, torch.bfloat16)
        assert bool((out[at[n]:] == 7).all())
    for bad, (i, r, most) in enumerate(((2, 99, None), (2, -1, None), (3, ids[3], 200))):
        out, err = torch.full_like(q, 7.0), i32([0])
        ids2 = list(ids)
        ids2[i] = r
        run_paged(q, kc, vc, tables, lens, new, ids2, out, err, max_kv=most, single=single)
        assert int(err) & 1
        assert bool((out[at[i]:at[i + 1]] == 7).all())
        rest = torch.ones(q.shape[0], dtype=torch.bool, device=DEV)
        rest[at[i]:at[i + 1]] = False
        check_attention(out[rest], *[x[rest] for x in ref], max(lens), 128, torch.bfloat16)


@pytest.mark.parametrize("single", [False, True])
def test_paged_attention_rows_that_see_nothing(single):
    """A request shorter than its new tokens: the tokens before its first
    position see nothing and get zeros."""
    new, ctx = ([1, 1], [5, 30]) if single else ([40, 3], [0, 30])
    q, kc, vc, tables, lens, ids = paged_case(new, ctx, 8, 2, 128, torch.float16, 16, 3)
    lens[ids[0]] = 0 if single else 25
    out = run_paged(q, kc, vc, tables, lens, new, ids, single=single)
    ref = paged_reference(q, kc, vc, tables, lens, new, ids, 128 ** -0.5)
    check_attention(out, *ref, max(lens), 128, torch.float16)
    assert bool((out[:1 if single else 15] == 0).all())


@pytest.mark.parametrize("single", [False, True])
def test_paged_attention_flags_a_bad_page(single):
    """A page outside the cache reads as zeros and sets the error word."""
    new = [1, 1] if single else [9, 20]
    q, kc, vc, tables, lens, ids = paged_case(new, [200, 300], 4, 1, 128, torch.bfloat16, 64, 6, junk=0.0)
    for bad in (-1, kc.shape[0], (1 << 31) - 1):
        t2 = tables.clone()
        t2[ids[1], 2] = bad
        err = i32([0])
        out = run_paged(q, kc, vc, t2, lens, new, ids, err=err, single=single)
        assert int(err) & 1
        k2, v2, t3 = kc.clone(), vc.clone(), tables
        k2[tables[ids[1], 2].long()] = 0
        v2[tables[ids[1], 2].long()] = 0
        ref = paged_reference(q, k2, v2, t3, lens, new, ids, 128 ** -0.5)
        check_attention(out, *ref, max(lens), 128, torch.bfloat16)


@pytest.mark.parametrize("op", ["packed", "chunk", "single"])
def test_attention_in_a_graph_reads_the_lengths_at_replay(op):
    """One capture, replayed on other lengths, another stream's eager call in
    between; two graphs of the same call do not disturb one another."""
    ops = _native.ops()
    hq, hkv, d, dtype, page = 8, 2, 128, torch.bfloat16, 32
    scale = d ** -0.5
    new = [1] * 4 if op == "single" else [30, 1, 200, 9]
    ctx = [900, 3, 5000, 64]
    q, kc, vc, tables, lens, ids = paged_case(new, ctx, hq, hkv, d, dtype, page, 21)
    n = sum(new)
    _, k, v = rows(n, hq, hkv, d, dtype, 22, False)
    cu, kv = i32(starts(new)), i32(lens)
    outs = [torch.zeros_like(q) for _ in range(2)]

    def call(out):
        if op == "packed":
            ops.packed_attention(q, k, v, cu, None, out, scale, None)
        else:
            ops.paged_attention(q, kc, vc, tables, kv, None if op == "single" else cu, i_ids, out,
                                max(lens), scale, None)

    def reference(new_, lens_):
        if op == "packed":
            return packed_reference(q, k, v, new_, None, scale)
        return paged_reference(q, kc, vc, tables, lens_, new_, ids, scale)

    i_ids = i32(ids)
    call(outs[0])
    torch.cuda.synchronize()
    graphs = []
    for out in outs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(out)
        graphs.append(g)
    changes = [(new, lens)]
    shorter = [max(m, x - 700) for m, x in zip([new[ids.index(r)] for r in range(4)], lens)]
    changes.append((new if op == "single" else [9, 200, 30, 1], lens if op == "packed" else [max(x, 200) for x in shorter]))
    for new_, lens_ in changes:
        lens_ = [min(a, b) for a, b in zip(lens_, lens)] if op != "packed" else lens_
        cu.copy_(i32(starts(new_)))
        kv.copy_(i32(lens_))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        third = torch.zeros_like(q)
        with torch.cuda.stream(side):
            call(third)
        for g in graphs:
            g.replay()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        ref = reference(new_, lens_)
        for out in (*outs, third):
            check_attention(out, *ref, max(max(lens), n), d, dtype)


def test_attention_repeats_bit_for_bit():
    """The same call gives the same bits, split over the keys or not."""
    new, ctx = [5, 1, 64], [6000, 12000, 300]
    q, kc, vc, tables, lens, ids = paged_case(new, ctx, 8, 2, 128, torch.bfloat16, 64, 31)
    a = run_paged(q, kc, vc, tables, lens, new, ids)
    for _ in range(3):
        assert torch.equal(a, run_paged(q, kc, vc, tables, lens, new, ids))


# ------------------------------------------------------- append and tables
@pytest.mark.parametrize("n,hkv,d,page,dtype,fused", [
    (1, 8, 128, 16, torch.bfloat16, True), (37, 3, 64, 5, torch.float16, False),
    (700, 1, 128, 64, torch.float16, True), (129, 12, 64, 128, torch.bfloat16, True)])
def test_paged_append(n, hkv, d, page, dtype, fused):
    """Rows to their slots, holes skipped, everything else as it was; with row
    ids and a device count; and zeros."""
    ops = _native.ops()
    pages = n // page + 3
    _, k, v = rows(n, 2, hkv, d, dtype, n, fused)
    g = torch.Generator().manual_seed(n)
    slots = torch.randperm(pages * page, generator=g)[:n]
    slots[::7] = -1
    kc = torch.full((pages, hkv, page, d), 3.0, dtype=dtype, device=DEV)
    vc = kc.clone()
    err = i32([0])

    def expect(rows_, src_k, src_v, ek, ev):
        for i, m in rows_:
            s = int(slots[m])
            if s >= 0:
                ek[s // page, :, s % page] = src_k[i] if src_k is not None else 0
                ev[s // page, :, s % page] = src_v[i] if src_v is not None else 0

    ek, ev = kc.clone(), vc.clone()
    ops.paged_append(k, v, slots.to(DEV), None, None, kc, vc, err)
    expect([(i, i) for i in range(n)], k, v, ek, ev)
    assert torch.equal(kc, ek) and torch.equal(vc, ev)
    ids = torch.randperm(n, generator=g)
    live = n // 2
    kc.fill_(3.0), vc.fill_(3.0)
    ek, ev = kc.clone(), vc.clone()
    ops.paged_append(k, v, slots.to(DEV), ids.to(torch.int32).to(DEV), i32([live]), kc, vc, err)
    expect([(i, int(ids[i])) for i in range(live)], k, v, ek, ev)
    assert torch.equal(kc, ek) and torch.equal(vc, ev)
    ops.paged_append(None, None, slots.to(DEV), None, None, kc, vc, err)
    expect([(i, i) for i in range(n)], None, None, ek, ev)
    assert torch.equal(kc, ek) and torch.equal(vc, ev) and int(err) == 0


def test_paged_append_flags_slots_and_rows_outside():
    ops = _native.ops()
    _, k, v = rows(4, 2, 2, 128, torch.float16, 1)
    kc = torch.zeros(2, 2, 16, 128, dtype=torch.float16, device=DEV)
    vc = kc.clone()
    for slots, ids in (([0, 32, 5, -1], None), ([0, -2, 5, -1], None), ([0, 1 << 40, 5, -1], None),
                       ([0, 7, 5, -1], [0, 4, 2, 3]), ([0, 7, 5, -1], [0, -1, 2, 3])):
        kc.zero_(), vc.zero_()
        err = i32([0])
        ops.paged_append(k, v, torch.tensor(slots, device=DEV), None if ids is None else i32(ids), None,
                         kc, vc, err)
        assert int(err) & 1
        want = torch.zeros_like(kc)
        want[0, :, 0], want[0, :, 5] = k[0], k[2]
        assert torch.equal(kc, want)


def run_tables(ctx, new, done, free, n_free, tables, page, n_slots, in_place=False):
    ops = _native.ops()
    c, f, nf, t = i32(ctx), i32(free), i32([n_free]), i32(tables)
    kv = c if in_place else torch.full_like(c, -7)
    nfo = nf if in_place else i32([-7])
    cu = torch.full((len(ctx) + 1,), -7, dtype=torch.int32, device=DEV)
    slots = torch.full((n_slots,), -7, dtype=torch.int64, device=DEV)
    pos = slots.clone()
    err = i32([0])
    ops.page_tables(c, i32(new), None if done is None else i32(done), f, nf, t, page, nfo, kv, cu,
                    slots, pos, err)
    return dict(free=f.tolist(), n_free=int(nfo), tables=t.tolist(), kv=kv.tolist(), cu=cu.tolist(),
                slots=slots.tolist(), pos=pos.tolist()), int(err)


@pytest.mark.parametrize("n,top,page,seed,in_place", [
    (1, 1, 16, 0, False), (5, 40, 7, 1, True), (300, 1, 64, 2, True), (700, 30, 16, 3, False),
    (40, 900, 128, 4, True), (1500, 3, 1, 5, False)])
def test_page_tables_over_steps(n, top, page, seed, in_place):
    """Steps of a serving loop against the reference: requests come, grow, end
    and are replaced; the page ids handed out stay distinct."""
    r = random.Random(seed)
    width = -(-(top * 6 + 20) // page)
    n_pages = n * width * 2 // 3 + 1
    free = list(range(n_pages))
    r.shuffle(free)
    n_free, ctx, tables = n_pages, [0] * n, [[-1] * width for _ in range(n)]
    for step in range(6):
        done = [int(ctx[i] > 0 and r.random() < 0.3) for i in range(n)] if step else None
        new = [r.randint(0, top) for _ in range(n)]
        cap = sum(new) + r.randint(0, 9)
        got, err = run_tables(ctx, new, done, free, n_free, tables, page, cap, in_place)
        want = page_tables_reference(ctx, new, done, free, n_free, tables, page, cap)
        for key in want:
            assert got[key] == want[key], (step, key)
        assert bool(err & 8) == (want["kv"] != [(0 if done and done[i] else ctx[i]) + new[i] for i in range(n)])
        ctx, free, n_free, tables = want["kv"], want["free"], want["n_free"], want["tables"]
        held = [p for i in range(n) for p in tables[i][:-(-ctx[i] // page)]] + free[:n_free]
        assert sorted(held) == list(range(n_pages))


def test_page_tables_many_tokens_and_long_requests():
    """A batch large enough for the cluster, one request of 70000 tokens."""
    ctx, new, page = [0, 13, 4000], [70000, 5000, 1], 16
    width = 4400
    n_pages = 5000
    tables = [[-1] * width, [0] + [-1] * (width - 1), list(range(1, 251)) + [-1] * (width - 250)]
    free = list(range(251, n_pages)) + [0] * 251
    got, err = run_tables(ctx, new, [0, 0, 1], free, n_pages - 251, tables, page, 80000)
    want = page_tables_reference(ctx, new, [0, 0, 1], free, n_pages - 251, tables, page, 80000)
    assert err == 0
    for key in want:
        assert got[key] == want[key], key


def test_page_tables_reports_what_does_not_fit():
    """Too few pages, a table too narrow, tokens past the slot map, negative
    lengths and a bad free count."""
    t = [[-1] * 2 for _ in range(3)]
    got, err = run_tables([0, 0, 0], [5, 9, 3], None, [4, 5, 6], 3, t, 4, 20)
    want = page_tables_reference([0, 0, 0], [5, 9, 3], None, [4, 5, 6], 3, t, 4, 20)
    assert err == 8 and got == want and got["kv"] == [5, 0, 3]  # 9 > 8 positions of a table row
    got, err = run_tables([0, 0, 0], [5, 8, 3], None, [4, 5, 6], 3, t, 4, 20)
    assert err == 8 and got["kv"] == [5, 0, 0] and got["n_free"] == 1
    assert got["slots"][:5] == [24, 25, 26, 27, 20] and got["slots"][5:] == [-1] * 15
    got, err = run_tables([0, 0, 0], [2, 3, 1], None, [4, 5, 6], 3, t, 4, 4)
    assert err == 4 and got["kv"] == [2, 0, 0] and got["cu"] == [0, 2, 5, 6]
    assert got["slots"] == [24, 25, -1, -1] and got["pos"] == [0, 1, 0, 1]
    got, err = run_tables([-4, 0, 0], [1, -2, 1], None, [4, 5, 6], 7, t, 4, 4)
    assert err == 4 and got["kv"] == [1, 0, 1] and got["n_free"] == 1


def test_a_serving_loop_over_the_paged_cache():
    """The operators together as a serving loop uses them: a wave of prompts in
    chunks, then decode steps with requests that end and start, every step's
    attention against the keys and values kept in plain lists."""
    ops = _native.ops()
    hq, hkv, d, dtype, page, n_req, width, n_pages = 8, 2, 128, torch.bfloat16, 16, 6, 40, 120
    scale = d ** -0.5
    g = torch.Generator(device=DEV).manual_seed(77)
    kc = torch.full((n_pages, hkv, page, d), float("nan"), dtype=dtype, device=DEV)
    vc = kc.clone()
    lens, n_free = i32([0] * n_req), i32([n_pages])
    free = torch.randperm(n_pages, generator=torch.Generator().manual_seed(5)).to(torch.int32).to(DEV)
    tables = torch.full((n_req, width), -1, dtype=torch.int32, device=DEV)
    cu, err = i32([0] * (n_req + 1)), i32([0])
    hist = [[torch.zeros(0, hkv, d, dtype=dtype, device=DEV)] * 2 for _ in range(n_req)]
    steps = [([100, 1, 33, 0, 260, 16], None), ([50, 40, 0, 128, 1, 16], None)] + \
        [([1, 1, 1, 1, 1, 1], None)] * 3 + [([1, 300, 1, 0, 1, 1], [0, 1, 0, 1, 0, 0])] + \
        [([1, 1, 1, 7, 1, 1], None)]
    for new, done in steps:
        n = sum(new)
        slots = torch.empty(n + 4, dtype=torch.int64, device=DEV)
        pos = torch.empty_like(slots)
        ops.page_tables(lens, i32(new), None if done is None else i32(done), free, n_free, tables, page,
                        n_free, lens, cu, slots, pos, err)
        q = torch.randn(n, hq, d, generator=g, device=DEV).to(dtype)
        kn = torch.randn(n, hkv, d, generator=g, device=DEV).to(dtype)
        vn = torch.randn(n, hkv, d, generator=g, device=DEV).to(dtype)
        ops.paged_append(kn, vn, slots, None, None, kc, vc, err)
        out = torch.empty_like(q)
        single = new == [1] * n_req
        ops.paged_attention(q, kc, vc, tables, lens, None if single else cu, None, out, 620, scale, err)
        a = 0
        for r, m in enumerate(new):
            if done and done[r]:
                hist[r] = [hist[r][0][:0], hist[r][1][:0]]
            hist[r] = [torch.cat([hist[r][0], kn[a:a + m]]), torch.cat([hist[r][1], vn[a:a + m]])]
            a += m
        L = lens.tolist()
        assert L == [h[0].shape[0] for h in hist] and int(err) == 0
        for r in range(n_req):
            assert torch.equal(gather_pages(kc, tables[r], L[r]), hist[r][0])
            assert torch.equal(gather_pages(vc, tables[r], L[r]), hist[r][1])
        ref = paged_reference(q, kc, vc, tables, L, new, list(range(n_req)), scale)
        check_attention(out, *ref, max(L), d, dtype)
