"""The paged cache in 4 bits on the GPU: the append with the heads' norms and the
position rotation, reading back, and attention, against 64-bit references.

What is held is compared bit by bit: the codes follow from the rows by rules with
one result, and the rotation that comes before is made in 64 bits on both sides.
The bound of the rotated queries is derived at its test, that of the attention in
ragged_helpers (the values that the cache holds are exact in the rows' type)."""
import random

import pytest
import torch

from tests import q4_helpers as Q
from tests.ragged_helpers import check_attention, paged_reference
from tests.test_gpu_ragged import i32, paged_case, rows, starts
from tide_b200 import _native

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16
HEADS = [(8, 2, 128, BF), (4, 4, 64, HF), (14, 2, 128, HF), (6, 2, 64, BF), (32, 1, 128, BF), (3, 3, 64, BF)]


def inv_freq(d, base=500000.0):
    return (1.0 / base ** (torch.arange(0, d, 2, device=DEV).double() / d)).float()


def append(q, k, v, slots, cache, ids=None, live=None, positions=None, freq=None, scaling=1.0, qw=None,
           kw=None, eps=1e-6, q_out=None, err=None):
    if q is not None and q_out is None:
        q_out = torch.empty(q.shape, dtype=q.dtype, device=DEV)
    _native.ops().paged_append_q4(q, k, v, slots, ids, live, positions, freq, scaling, qw, kw, eps, q_out,
                                  cache, err)
    return q_out


def read(cache, slots, dtype, err=None, fill=0.0):
    d = cache.shape[3] // 18
    k = torch.full((slots.numel(), cache.shape[1], d), fill, dtype=dtype, device=DEV)
    v = k.clone()
    _native.ops().paged_read_q4(cache, slots, k, v, err)
    return k, v


def empty_cache(pages, hkv, page, d, fill=0):
    return torch.full((pages, hkv, page // 16, 18 * d), fill, dtype=torch.uint8, device=DEV)


def check_q(out, ref, size, dtype, d):
    """Rounded once to dtype (eps / 2), from 32-bit terms: the head's sum of squares
    (d adds of 2^-24, halved by the root), the root (2^-22), two products (2^-24
    each), cosine and sine (2^-24), a product and a sum of the rotation."""
    rel = (d / 2 + 4 + 2 + 1 + 2) * 2.0 ** -24
    may = torch.finfo(dtype).eps / 2 * (ref.abs() + rel * size) + rel * size + torch.finfo(dtype).tiny
    off = (out.double() - ref).abs()
    assert bool((off <= may).all()), (off / may).max().item()


# ----------------------------------------------------------- append, read
@pytest.mark.parametrize("hq,hkv,d,dtype", HEADS)
@pytest.mark.parametrize("n", [1, 5, 300, 2500])
@pytest.mark.parametrize("norm,rotate", [(True, True), (False, True), (True, False), (False, False)])
def test_append(hq, hkv, d, dtype, n, norm, rotate):
    page = 48
    q, k, v = rows(n, hq, hkv, d, dtype, n + hq, True)
    g = torch.Generator(device=DEV).manual_seed(n)
    pages = n // page + 3
    slots = torch.randperm(pages * page, generator=g, device=DEV)[:n]
    slots[n // 2] = -1 if n > 1 else slots[n // 2]
    pos = torch.randint(0, 200000, (n,), generator=g, device=DEV)
    pos[0] = 0
    w = [(1 + 0.3 * torch.randn(d, generator=g, device=DEV)).to(dtype) if norm else None for _ in range(2)]
    freq = inv_freq(d) if rotate else None
    cache = empty_cache(pages, hkv, page, d, 0xA5)
    before = cache.clone()
    err = i32([0])
    out = append(q, k, v, slots, cache, positions=pos if rotate else None, freq=freq, qw=w[0], kw=w[1], err=err)
    assert int(err) == 0
    check_q(out, *Q.turned(q, pos, freq, w[0], 1e-6), dtype, d)
    real = slots >= 0
    kf = Q.turned(k, pos, freq, w[1], 1e-6)[0].float()
    got = read(cache, slots, dtype)
    for x, y in zip(got, (kf, v)):
        assert torch.equal(x[real].double(), Q.values(y, dtype)[real])
        assert bool((x[~real] == 0).all())
    # and nothing else of the cache has changed
    at = torch.zeros(pages * page, dtype=torch.bool, device=DEV)
    at[slots[real]] = True
    mine = Q.token_bytes(at.view(pages, page), hkv, d)
    assert torch.equal(cache[~mine], before[~mine])
    dense = [torch.zeros(pages * page, hkv, d, dtype=torch.float64, device=DEV) for _ in range(2)]
    for x, y in zip(dense, (kf, v)):
        x[slots[real]] = y[real].double()
    whole = Q.pack(*[x.view(pages, page, hkv, d).transpose(1, 2) for x in dense], dtype)
    assert torch.equal(cache[mine], whole[mine])


@pytest.mark.parametrize("dtype", [BF, HF])
def test_append_of_odd_groups(dtype):
    """Groups of one sign, of zeros, of one value, of tiny numbers, next to the
    largest numbers, and of values halfway between two codes (ties to even)."""
    n, d = 64, 128
    g = torch.Generator(device=DEV).manual_seed(1)
    k = torch.randn(n, 1, d, generator=g, device=DEV)
    k[0], k[1], k[2] = k[0].abs(), -k[1].abs(), 0
    k[3] = 0.37
    k[4] = k[4] * 1e-7
    k[5] = torch.finfo(dtype).max * torch.sign(k[5])
    k[6] = torch.finfo(dtype).max
    k[7, :, 32:64] = 0
    k[8:40] = torch.randint(-15, 16, (32, 1, d), generator=g, device=DEV) / 2 * \
        torch.randint(8, 16, (32, 1, 1), generator=g, device=DEV) / 8
    k[40:] = k[40:] * 10.0 ** torch.randint(-6, 4, (24, 1, 1), generator=g, device=DEV)
    k = k.to(dtype)
    v = k.flip(0).contiguous()
    cache = empty_cache(4, 1, 16, d)
    slots = torch.arange(n, device=DEV).flip(0).contiguous()
    append(None, k, v, slots, cache)
    for x, y in zip(read(cache, slots, dtype), (k, v)):
        assert bool(x.isfinite().all())
        assert torch.equal(x.double(), Q.values(y, dtype))


@pytest.mark.parametrize("dtype", [BF, HF])
def test_a_group_with_a_value_that_is_not_finite_reads_as_nan(dtype):
    k = torch.randn(3, 2, 64, device=DEV).to(dtype)
    v = torch.randn(3, 2, 64, device=DEV).to(dtype)
    k[1, 0, 40] = float("nan")
    v[2, 1, 3] = float("-inf")
    cache = empty_cache(1, 2, 16, 64)
    slots = torch.tensor([3, 9, 15], device=DEV)
    append(None, k, v, slots, cache)
    gk, gv = read(cache, slots, dtype)
    for x, y in ((gk, k), (gv, v)):
        odd = ~y.unflatten(-1, (2, 32)).isfinite().all(-1, keepdim=True).expand(3, 2, 2, 32).flatten(-2)
        assert bool(x[odd].isnan().all())
        assert torch.equal(x[~odd].double(), Q.values(y, dtype)[~odd])


def test_append_rows_of_a_slot_map_live_counts_and_zeros():
    """Surviving rows among a step's tokens: zeros to every slot, then the rows, of
    which the device's count are live."""
    n, hq, hkv, d, dtype, page = 40, 8, 2, 128, BF, 16
    q, k, v = rows(n, hq, hkv, d, dtype, 7, False)
    slots = torch.randperm(5 * page, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)[:n + 8]
    slots[3] = -1
    pos = torch.arange(n + 8, device=DEV) * 37
    ids = torch.randperm(n + 8, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV)[:n].int()
    cache = empty_cache(5, hkv, page, d, 0xFF)
    out = torch.full_like(q, 7.0)
    _native.ops().paged_append_q4(None, None, None, slots, None, None, None, None, 1.0, None, None, 0.0, None,
                                  cache, None)
    append(q, k, v, slots, cache, ids, i32([29]), pos, inv_freq(d), 1.25, q_out=out)
    ref, size = Q.turned(q, pos[ids.long()], inv_freq(d), None, 0.0, 1.25)
    check_q(out[:29], ref[:29], size[:29], dtype, d)
    assert bool((out[29:] == 7).all())
    gk, gv = read(cache, slots, dtype, fill=5.0)
    mine = torch.zeros(n + 8, dtype=torch.bool, device=DEV)
    mine[ids[:29].long()] = True
    none = slots < 0
    assert bool((gk[none] == 5).all()) and bool((gk[~mine & ~none] == 0).all()) and \
        bool((gv[~mine & ~none] == 0).all())
    kf = Q.turned(k, pos[ids.long()], inv_freq(d), None, 0.0, 1.25)[0].float()
    live = ids[:29].long()
    keep = ~none[live]
    assert torch.equal(gk[live][keep].double(), Q.values(kf, dtype)[:29][keep])
    assert torch.equal(gv[live][keep].double(), Q.values(v, dtype)[:29][keep])


def test_append_and_read_flag_places_outside_the_cache():
    k = torch.randn(4, 1, 64, device=DEV).to(HF)
    cache = empty_cache(2, 1, 16, 64, 0xA5)
    for slots, ids in ((torch.tensor([1, 32, -2, 5], device=DEV), None),
                       (torch.tensor([1, 5], device=DEV), i32([0, 2, -1, 1]))):
        c, err = cache.clone(), i32([0])
        q_out = torch.full_like(k, 7.0)
        append(k, k, k, slots, c, ids, q_out=q_out, err=err)
        assert int(err) == 1
        at = torch.zeros(2, 16, dtype=torch.bool, device=DEV)
        at[0, 1] = at[0, 5] = True
        assert torch.equal(c[~Q.token_bytes(at, 1, 64)], cache[~Q.token_bytes(at, 1, 64)])
        gk, _ = read(c, torch.tensor([1, 5], device=DEV), HF)
        assert torch.equal(gk.double(), Q.values(k[[0, 3]], HF))
        # (a row id outside has no position, so its query is left)
        assert torch.equal(q_out[[0, 3]], k[[0, 3]])
        assert bool((q_out[[1, 2]] == 7).all()) == (ids is not None)
    err = i32([0])
    gk, _ = read(cache, torch.tensor([0, 32, -5], device=DEV), HF, err, 3.0)
    assert int(err) == 1 and bool((gk[1:] == 3).all())


def test_operators_refuse_what_does_not_fit():
    ops = _native.ops()
    cache = empty_cache(2, 2, 16, 64)
    k = torch.zeros(3, 2, 64, dtype=HF, device=DEV)
    slots = torch.arange(3, device=DEV)
    freq = inv_freq(64)

    def bad(**kw):
        a = dict(q=None, k=k, v=k, slots=slots, ids=None, live=None, pos=None, freq=None, scaling=1.0,
                 qw=None, kw=None, eps=0.0, out=None, cache=cache, err=None)
        a.update(kw)
        with pytest.raises(RuntimeError):
            ops.paged_append_q4(*a.values())

    bad(v=None)
    bad(q=k)
    bad(q=k, k=None, v=None, out=k.clone())
    bad(freq=freq)
    bad(freq=freq, pos=slots[:2])
    bad(freq=freq, pos=slots.int())
    bad(freq=freq[:31], pos=slots)
    bad(freq=freq.half(), pos=slots)
    bad(kw=torch.ones(64, dtype=BF, device=DEV))
    bad(kw=torch.ones(63, dtype=HF, device=DEV))
    bad(slots=slots[:2])
    bad(slots=slots.int())
    bad(k=k[:, :1], v=k[:, :1])
    bad(k=k.expand(3, 2, 64)[:, :, :32], v=k)
    bad(k=k.float(), v=k.float())
    bad(cache=cache.view(torch.int8))
    bad(cache=cache[:, :, :, :100])
    bad(cache=cache[:, :1])
    with pytest.raises(RuntimeError):
        ops.paged_read_q4(cache, slots, k, k[:2], None)
    with pytest.raises(RuntimeError):
        ops.paged_read_q4(cache, slots, k.float(), k.float(), None)
    with pytest.raises(RuntimeError):
        ops.paged_attention_q4(k, empty_cache(2, 2, 16, 128), i32([[0]]), i32([1]), i32([0, 3]), None,
                               k.clone(), 16, 0.1, None)
    with pytest.raises(RuntimeError):
        ops.paged_attention_q4(k, cache, i32([[0]]), i32([1]), i32([0, 3]), None, k.clone(), 17, 0.1, None)


# -------------------------------------------------------------- attention
def q4_case(new, ctx, hq, hkv, d, dtype, page, seed, n_req=None):
    """paged_case with its caches in 4 bits: those, and dense ones with the values
    that they hold.  Unused places are bytes of ones, which read as NaN."""
    q, kc, vc, tables, lens, ids = paged_case(new, ctx, hq, hkv, d, dtype, page, seed, n_req)
    used = kc.isfinite().all(-1).all(1)
    clean = [torch.where(used[:, None, :, None], x, 0) for x in (kc, vc)]
    cache = torch.full((kc.shape[0], hkv, page // 16, 18 * d), 0xFF, dtype=torch.uint8, device=DEV)
    Q.pack(*clean, dtype, cache, used)
    held = [Q.values(x, dtype).to(dtype) for x in clean]
    return q, cache, held, tables, lens, ids


def attend(q, cache, tables, lens, new, ids, max_kv=None, single=False, out=None, err=None, n_dev=None):
    out = torch.full_like(q, 7.0) if out is None else out
    most = max(lens) if max_kv is None else max_kv
    _native.ops().paged_attention_q4(q, cache, tables, i32(lens), None if single else i32(starts(new)),
                                     i32(ids), out, most, q.shape[2] ** -0.5, err, n_dev)
    return out


def check(out, q, held, tables, lens, new, ids):
    ref = paged_reference(q, *held, tables, lens, new, ids, q.shape[2] ** -0.5)
    check_attention(out, *ref, max(max(lens), 1), q.shape[2], q.dtype)


@pytest.mark.parametrize("hq,hkv,d,dtype", HEADS + [(16, 1, 128, HF), (64, 1, 64, HF), (40, 1, 128, BF)])
@pytest.mark.parametrize("ctx,page", [([0], 16), ([0, 1, 15, 16, 17, 300, 33], 16), ([700, 2, 63], 64),
                                      ([4500], 32)], ids=str)
def test_attention_of_single_tokens(hq, hkv, d, dtype, ctx, page):
    new = [1] * len(ctx)
    q, cache, held, tables, lens, ids = q4_case(new, ctx, hq, hkv, d, dtype, page, hq + len(ctx), len(ctx) + 1)
    err = i32([0])
    out = attend(q, cache, tables, lens, new, ids, single=True, err=err)
    assert int(err) == 0
    check(out, q, held, tables, lens, new, ids)
    # as packed sequences of one token they are the same call
    check(attend(q, cache, tables, lens, new, ids), q, held, tables, lens, new, ids)


@pytest.mark.parametrize("hq,hkv,d,dtype", HEADS + [(64, 1, 64, HF)])
@pytest.mark.parametrize("new,ctx,page", [([2, 0, 5, 1], [0, 40, 700, 3], 16), ([9, 1, 7], [2000, 0, 33], 32),
                                          ([130, 3], [5, 260], 64), ([1, 300, 40], [900, 20, 128], 128),
                                          ([33], [1], 16)], ids=str)
def test_attention_of_chunks(hq, hkv, d, dtype, new, ctx, page):
    q, cache, held, tables, lens, ids = q4_case(new, ctx, hq, hkv, d, dtype, page, sum(new) + hq)
    err = i32([0])
    out = attend(q, cache, tables, lens, new, ids, err=err)
    assert int(err) == 0
    check(out, q, held, tables, lens, new, ids)


@pytest.mark.parametrize("new", [[1, 1, 1], [3, 1, 2], [40, 70, 1]], ids=str)
def test_attention_under_a_wide_bound(new):
    """max_kv_len far above the lengths: splits and rounds that find no keys."""
    hq, hkv, d, dtype = 8, 4, 128, BF
    q, cache, held, tables, lens, ids = q4_case(new, [5, 100, 30], hq, hkv, d, dtype, 16, 9)
    wide = torch.cat([tables, torch.full((3, 200000 // 16), -1, dtype=torch.int32, device=DEV)], 1).contiguous()
    for most in (1000, 200000):
        out = attend(q, cache, wide, lens, new, ids, most, single=max(new) == 1)
        check(out, q, held, tables, lens, new, ids)


@pytest.mark.parametrize("single", [True, False])
@pytest.mark.parametrize("named", [True, False])
def test_attention_in_rounds(single, named):
    """More 16-bit pages than a round of the many-rows path may have (40 query heads
    on one KV head take it for single tokens too), with and without named requests
    and a live count from the device."""
    hq, hkv, d, dtype, B = 40, 1, 128, BF, 37
    new = [1] * B if single else [1 + i % 5 for i in range(B)]
    q, cache, held, tables, lens, ids = q4_case(new, [7 * i for i in range(B)], hq, hkv, d, dtype, 16, 12)
    wide = torch.cat([tables, torch.full((B, 200000 // 16), -1, dtype=torch.int32, device=DEV)], 1).contiguous()
    if not named:
        wide, lens = wide[ids].contiguous(), [lens[r] for r in ids]
        tables, ids = tables[ids], list(range(B))
    for live in (None, 30, 0):
        out, err = torch.full_like(q, 7.0), i32([0])
        _native.ops().paged_attention_q4(q, cache, wide, i32(lens), None if single else i32(starts(new)),
                                         i32(ids) if named else None, out, 200000, d ** -0.5, err,
                                         None if live is None else i32([live]))
        n = B if live is None else live
        at = starts(new)[n]
        assert int(err) == 0 and bool((out[at:] == 7).all())
        if n:
            check(out[:at], q[:at], held, tables, lens, new[:n], ids[:n])


@pytest.mark.parametrize("new", [[1, 1], [3, 2], [150, 20]], ids=str)
def test_attention_flags_bad_pages_and_requests(new):
    hq, hkv, d, dtype = 4, 2, 128, HF
    q, cache, held, tables, lens, ids = q4_case(new, [100, 70], hq, hkv, d, dtype, 16, 3)
    single = max(new) == 1
    broken = tables.clone()
    broken[ids[0], 2] = cache.shape[0]
    err = i32([0])
    out = attend(q, cache, broken, lens, new, ids, single=single, err=err)
    assert int(err) & 1
    held0 = [torch.cat([x, torch.zeros_like(x[:1])]) for x in held]
    check(out, q, held0, broken, lens, new, ids)  # (reads as zeros)
    for bad_lens, bad_ids in ((lens, [5, ids[1]]), ([lens[0] + 5000 if r == ids[0] else lens[r] for r in (0, 1)], ids)):
        err.zero_()
        out = attend(q, cache, tables, bad_lens, new, bad_ids, max(lens), single=single, err=err)
        assert int(err) & 1 and bool((out[:new[0]] == 7).all())
        check(out[new[0]:], q[new[0]:], held, tables, lens, new[1:], ids[1:])


@pytest.mark.parametrize("new", [[1, 1], [4, 2], [90, 20]], ids=str)
def test_attention_of_groups_that_are_not_finite(new):
    """A value group that is NaN reaches the tokens that see it, and no others; so
    does a key."""
    hq, hkv, d, dtype, page = 4, 2, 64, BF, 16
    q, cache, held, tables, lens, ids = q4_case(new, [100, 70], hq, hkv, d, dtype, page, 5)
    clean = attend(q, cache, tables, lens, new, ids)
    r = ids[0]
    for side, pos in ((1, lens[r] - 1), (1, 50), (0, lens[r] - 1)):
        c = cache.clone()
        pg, blk, t = int(tables[r, pos // page]), pos % page // 16, pos % 16
        at = 16 * d + side * d + 2 * (16 + t % 4 * 4 + t // 4)  # the second group of channels
        c[pg, 1, blk, at], c[pg, 1, blk, at + 1] = 0xC0, 0x7F
        out = attend(q, c, tables, lens, new, ids)
        sees = torch.zeros(q.shape[0], dtype=torch.bool, device=DEV)
        sees[:new[0]] = torch.arange(new[0], device=DEV) + lens[r] - new[0] >= pos
        mask = torch.zeros_like(out, dtype=torch.bool)
        mask[sees, 2:, 32 if side else 0:] = True
        assert bool(out[mask].isnan().all())
        assert torch.equal(out[~mask], clean[~mask])


def test_attention_of_strided_rows_and_a_count_from_the_device():
    hq, hkv, d, dtype = 8, 2, 128, BF
    new = [1] * 9
    q, cache, held, tables, lens, ids = q4_case(new, [50 * i for i in range(9)], hq, hkv, d, dtype, 32, 6)
    big = torch.zeros(9, hq * d + 256, dtype=dtype, device=DEV)
    big[:, 128:128 + hq * d] = q.view(9, -1)
    qs = big[:, 128:128 + hq * d].view(9, hq, d)
    out, err = torch.full_like(q, 7.0), i32([0])
    attend(qs, cache, tables, lens, new, ids, single=True, out=out, err=err, n_dev=i32([6]))
    check(out[:6], q[:6], held, tables, lens, new[:6], ids[:6])
    assert bool((out[6:] == 7).all()) and int(err) == 0
    attend(qs, cache, tables, lens, new, ids, single=True, out=out, err=err, n_dev=i32([10]))
    assert int(err) & 4
    check(out, q, held, tables, lens, new, ids)


def test_the_same_request_twice():
    """Two sequences of one request (two branches that share their past)."""
    hq, hkv, d, dtype = 4, 2, 128, BF
    q, cache, held, tables, lens, ids = q4_case([2, 3], [300, 40], hq, hkv, d, dtype, 16, 8)
    for new in ([1, 1, 1], [2, 2, 1], [60, 80, 33]):
        twice = [ids[0], ids[0], ids[1]]
        x = torch.randn(sum(new), hq, d, device=DEV).to(dtype)
        new = [min(n, lens[r]) for n, r in zip(new, twice)]
        x = x[:sum(new)].contiguous()
        out = attend(x, cache, tables, lens, new, twice, single=max(new) == 1)
        check(out, x, held, tables, lens, new, twice)


def test_new_tokens_that_see_no_key_get_zeros():
    """More new tokens than the request has positions."""
    hq, hkv, d, dtype = 4, 2, 128, HF
    q, cache, held, tables, lens, ids = q4_case([3], [4], hq, hkv, d, dtype, 16, 8)
    for n in (9, 70):
        x = torch.randn(n, hq, d, device=DEV).to(dtype)
        out = attend(x, cache, tables, lens, [n], ids)
        assert bool((out[:n - 7] == 0).all())
        check(out[n - 7:], x[n - 7:], held, tables, lens, [7], ids)
    out = attend(x[:2].contiguous(), cache, tables, [0], [1, 1], [0, 0], 16, single=True)
    assert bool((out == 0).all())


# ---------------------------------------------------------------- together
@pytest.mark.parametrize("graph", [False, True])
def test_a_step_after_another(graph):
    """Page tables, append and attention of several steps, the requests' lengths on
    the device alone, as one captured step replayed, on a stream of its own."""
    B, hq, hkv, d, dtype, page, width = 5, 8, 2, 128, BF, 16, 8
    r = random.Random(2)
    ctx0 = [r.randint(0, 40) for _ in range(B)]
    ops = _native.ops()
    pages = B * width
    cache = empty_cache(pages, hkv, page, d)
    free = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).int().to(DEV)
    n_free, tables, lens = i32([pages]), i32([[-1] * width] * B), i32([0] * B)
    cu, err = i32([0] * (B + 1)), i32([0])
    freq = inv_freq(d, 10000.0)
    hist = [[[] for _ in range(B)] for _ in range(2)]

    def step(new, x, slots, pos, single):
        q, k, v = (t.view(x.shape[0], -1, d) for t in x.split([hq * d, hkv * d, hkv * d], 1))
        ops.page_tables(lens, new, None, free, n_free, tables, page, n_free, lens, cu, slots, pos, err)
        q_rot, out = torch.empty(q.shape, dtype=dtype, device=DEV), torch.empty(q.shape, dtype=dtype, device=DEV)
        ops.paged_append_q4(q, k, v, slots, None, None, pos, freq, 1.0, None, None, 0.0, q_rot, cache, err)
        ops.paged_attention_q4(q_rot, cache, tables, lens, None if single else cu, None, out, page * width,
                               d ** -0.5, err)
        return q_rot, out

    def expect(x, new, at0, q_rot, out):
        q, k, v = (t.reshape(x.shape[0], -1, d) for t in x.split([hq * d, hkv * d, hkv * d], 1))
        a = 0
        for b in range(B):
            n = new[b]
            pos = torch.arange(at0[b], at0[b] + n, device=DEV)
            kf = Q.turned(k[a:a + n], pos, freq, None, 0.0)[0].float()
            hist[0][b].append(Q.values(kf, dtype).to(dtype))
            hist[1][b].append(Q.values(v[a:a + n], dtype).to(dtype))
            if n:
                kk, vv = torch.cat(hist[0][b]), torch.cat(hist[1][b])
                m = kk.shape[0]
                dense = [torch.zeros(1, hkv, m, d, dtype=dtype, device=DEV) for _ in range(2)]
                dense[0][0], dense[1][0] = kk.transpose(0, 1), vv.transpose(0, 1)
                ref = paged_reference(q_rot[a:a + n], *dense, i32([[0]]), [m], [n], [0], d ** -0.5)
                check_attention(out[a:a + n], *ref, m, d, dtype)
            a += n

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        n0 = sum(ctx0)
        g = torch.Generator(device=DEV).manual_seed(3)
        x = torch.randn(n0, (hq + 2 * hkv) * d, generator=g, device=DEV).to(dtype)
        slots, pos = (torch.empty(n0, dtype=torch.int64, device=DEV) for _ in range(2))
        q_rot, out = step(i32(ctx0), x, slots, pos, False)
        expect(x, ctx0, [0] * B, q_rot, out)
        ones, buf = i32([1] * B), torch.empty(B, (hq + 2 * hkv) * d, dtype=dtype, device=DEV)
        slots, pos = (torch.empty(B, dtype=torch.int64, device=DEV) for _ in range(2))
        if graph:
            saved = [t.clone() for t in (lens, n_free, free, tables, cache)]
            step(ones, buf, slots, pos, True)
            for t, s in zip((lens, n_free, free, tables, cache), saved):
                t.copy_(s)
            torch.cuda.synchronize()
            cg = torch.cuda.CUDAGraph()
            with torch.cuda.graph(cg, stream=side):
                q_rot, out = step(ones, buf, slots, pos, True)
        for i in range(30):
            buf.copy_(torch.randn(buf.shape, generator=g, device=DEV))
            if graph:
                cg.replay()
            else:
                q_rot, out = step(ones, buf, slots, pos, True)
            expect(buf, [1] * B, [c + i for c in ctx0], q_rot, out)
    torch.cuda.current_stream().wait_stream(side)
    assert int(err) == 0


def test_attention_of_single_tokens_beside_a_prompt():
    """A batch whose calls need both kernels: many single tokens and one long chunk."""
    hq, hkv, d, dtype = 8, 2, 128, BF
    new = [1] * 40 + [300] + [2] * 20 + [0, 33]
    q, cache, held, tables, lens, ids = q4_case(new, [13 * i % 700 for i in range(len(new))], hq, hkv, d, dtype, 16, 4)
    for most in (max(lens), 5000):
        wide = torch.cat([tables, torch.full((len(new), 5000 // 16), -1, dtype=torch.int32, device=DEV)], 1).contiguous()
        err = i32([0])
        out = attend(q, cache, wide, lens, new, ids, most, err=err)
        assert int(err) == 0
        check(out, q, held, tables, lens, new, ids)


def test_attention_of_very_many_sequences():
    hq, hkv, d, dtype, B = 4, 1, 64, HF, 1500
    new = [i % 3 for i in range(B)]
    q, cache, held, tables, lens, ids = q4_case(new, [7 * i % 90 for i in range(B)], hq, hkv, d, dtype, 16, 2)
    for most in (max(lens), 600):
        wide = torch.cat([tables, torch.full((B, 600 // 16), -1, dtype=torch.int32, device=DEV)], 1).contiguous()
        check(attend(q, cache, wide, lens, new, ids, most), q, held, tables, lens, new, ids)
    single = [r for n, r in zip(new, ids) if n]
    x = torch.randn(len(single), hq, d, device=DEV).to(dtype)
    check(attend(x, cache, tables, lens, [1] * len(single), single, single=True), x, held, tables, lens,
          [1] * len(single), single)


def test_a_cache_past_4_gigabytes():
    """Pages whose bytes lie past 2^32: what a small cache gives."""
    hq, hkv, d, dtype, page = 8, 8, 128, BF, 64
    pages = 60000  # of 73728 bytes
    big = torch.empty(pages, hkv, page // 16, 18 * d, dtype=torch.uint8, device=DEV)
    place = torch.tensor([pages - 1, 58254, pages - 7], device=DEV)
    q, k, v = rows(150, hq, hkv, d, dtype, 3)
    at = torch.arange(150, device=DEV)
    slots = place[at // page] * page + at % page
    q_rot = append(q, k, v, slots, big, positions=at, freq=inv_freq(d))
    gk, gv = read(big, slots, dtype)
    kf = Q.turned(k, at, inv_freq(d), None, 0.0)[0].float()
    assert torch.equal(gk.double(), Q.values(kf, dtype)) and torch.equal(gv.double(), Q.values(v, dtype))
    held = [torch.zeros(3 * page, hkv, d, dtype=dtype, device=DEV) for _ in range(2)]
    held[0][:150], held[1][:150] = gk, gv
    held = [x.view(3, page, hkv, d).transpose(1, 2).contiguous() for x in held]
    tables = place.view(1, 3).int()
    for new in ([1], [20], [150]):
        x = q_rot[150 - new[0]:].contiguous()
        out = attend(x, big, tables, [150], new, [0], single=new == [1])
        check(out, x, held, torch.tensor([[0, 1, 2]], device=DEV), [150], new, [0])
    _native.ops().paged_append_q4(None, None, None, slots, None, None, None, None, 1.0, None, None, 0.0, None, big, None)
    assert not read(big, slots, dtype, fill=1.0)[0].any()


def test_a_captured_chunk_call_takes_other_lengths():
    """One captured call over tokens dealt to the sequences in several ways: all
    short, one long, one empty, which the two kernels share differently."""
    hq, hkv, d, dtype, B = 8, 2, 128, BF, 61
    n = 6 * B
    splits = [[6] * B, [1] * 30 + [n - 60] + [1] * 30, [n] + [0] * (B - 1), [0, 12] * 30 + [6]]
    _, cache, held, tables, lens, ids = q4_case([n] * B, [100 + 3 * i for i in range(B)], hq, hkv, d, dtype, 16, 5)
    most = max(lens)
    x = torch.randn(n, hq, d, device=DEV).to(dtype)
    cu, kv, out, err = i32([0] * (B + 1)), i32([0] * len(lens)), torch.zeros_like(x), i32([0])

    def call():
        _native.ops().paged_attention_q4(x, cache, tables, kv, cu, i32_ids, out, most, d ** -0.5, err)

    i32_ids = i32(ids)
    graph = None
    for new in splits + splits[:1]:
        cu.copy_(i32(starts(new)))
        mine = list(lens)
        for k, r in zip(new, ids):
            mine[r] = 90 + k
        kv.copy_(i32(mine))
        if graph is None:
            call()
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                call()
        out.fill_(7.0)
        graph.replay()
        assert int(err) == 0
        check(out, x, held, tables, mine, new, ids)


def test_calls_on_two_streams_do_not_meet():
    """Attention and appends of two caches at once, each on a stream of its own,
    against the same one after the other."""
    hq, hkv, d, dtype = 8, 2, 128, BF
    cases = [q4_case([1] * 40, [50 * i for i in range(40)], hq, hkv, d, dtype, 16, s) for s in (1, 2)]
    chunk = [q4_case([30, 90, 2], [900, 20, 500], hq, hkv, d, dtype, 32, s) for s in (3, 4)]
    streams = [torch.cuda.Stream() for _ in range(2)]

    def work(c, k):
        outs = []
        for q, cache, _, tables, lens, ids in (c, k):
            for _ in range(3):
                new = [1] * 40 if q.shape[0] == 40 else [30, 90, 2]
                outs.append(attend(q, cache, tables, lens, new, ids, max(lens),
                                   single=q.shape[0] == 40))
                kk = torch.full((5, hkv, d), 0.5, dtype=dtype, device=DEV)
                mine = empty_cache(2, hkv, 16, d)
                append(None, kk, kk, torch.arange(5, device=DEV), mine)
                outs.append(mine)
        return outs

    want = [work(c, k) for c, k in zip(cases, chunk)]
    torch.cuda.synchronize()
    got = []
    for s, c, k in zip(streams, cases, chunk):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(work(c, k))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


@pytest.mark.parametrize("dtype,x,scaling,finite", [
    (HF, 43648.0, 1.5, True), (HF, 43680.0, 1.5, False), (HF, -43680.0, 1.5, False), (HF, 65504.0, 2.0, False),
    (BF, 2.0 ** 127, 510 / 256, True), (BF, 2.0 ** 127, 511 / 256, False), (BF, 2.0 ** 127, 2.0, False)], ids=str)
def test_keys_that_the_rotation_takes_past_their_type(dtype, x, scaling, finite):
    """At position 0 the rotation is the scaling alone, exact here: keys that round
    to infinity in their type make their group NaN, the others are held."""
    n, hkv, d = 3, 2, 128
    _, k, v = rows(n, 2, hkv, d, dtype, 9)
    k[1, 1, 40] = x
    slots = torch.arange(n, device=DEV)
    cache = empty_cache(1, hkv, 16, d)
    append(None, k, v, slots, cache, positions=torch.zeros_like(slots), freq=torch.ones(d // 2, device=DEV),
           scaling=scaling)
    turned = k.double() * scaling
    if not finite:
        turned[1, 1, 40] = float("inf")
    got, values = read(cache, slots, dtype)
    odd = torch.zeros_like(got, dtype=torch.bool)
    odd[1, 1, 32:64] = not finite
    assert torch.equal(got.isnan(), odd) and bool(got.isfinite()[~odd].all())
    for y, want in ((got, turned), (values, v)):
        assert torch.equal(y.double().nan_to_num(0.5), Q.values(want, dtype).nan_to_num(0.5))
