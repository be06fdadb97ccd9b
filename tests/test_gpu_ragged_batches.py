"""The ragged operators on batches that take more than one of their kernels or
more than one round of the GPU: many sequences, keys past the L2, single
tokens beside long chunks, wide head groups, other streams, shared memory
pools, rows that are only 16-byte aligned."""
import random

import pytest
import torch

from tests.ragged_helpers import check_attention, packed_reference, paged_reference
from tests.test_gpu_ragged import i32, paged_case, rows, run_packed, run_paged, run_tables, starts
from tests.ragged_helpers import page_tables_reference
from tide_b200 import _native

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("n_seqs,top", [(1100, 9), (300, 200)])
def test_packed_attention_many_sequences(n_seqs, top):
    r = random.Random(n_seqs)
    lens = [r.randint(0, top) for _ in range(n_seqs)]
    q, k, v = rows(sum(lens), 4, 2, 64, torch.bfloat16, 1)
    zeros = i32([r.randint(-2, 50) for _ in range(sum(lens))])
    out = run_packed(q, k, v, lens, zeros)
    ref = packed_reference(q, k, v, lens, zeros.clamp(min=0), 64 ** -0.5)
    check_attention(out, *ref, top + 50, 64, torch.bfloat16)


def test_packed_attention_keys_past_the_l2():
    """100 MB of keys and values: several groups of sequences, more units than
    SMs, one sequence of a group's size by itself."""
    r = random.Random(2)
    lens = [r.randint(1, 900) for _ in range(60)] + [6000] + [r.randint(300, 700) for _ in range(24)]
    hkv, d = 4, 128
    assert sum(lens) * hkv * d * 4 > 80 << 20
    q, k, v = rows(sum(lens), hkv, hkv, d, torch.bfloat16, 2, False)
    out = run_packed(q, k, v, lens)
    at = starts(lens)
    for i in (0, 7, 30, 59, 60, 61, 70, 84):
        rows_ = slice(at[i], at[i + 1])
        ref = packed_reference(q[rows_], k[rows_], v[rows_], [lens[i]], None, d ** -0.5)
        check_attention(out[rows_], *ref, lens[i], d, torch.bfloat16)
    assert torch.isfinite(out.float()).all()
    assert torch.equal(out, run_packed(q, k, v, lens))


@pytest.mark.parametrize("hq,hkv,d,dtype", [(8, 2, 128, torch.bfloat16), (12, 4, 64, torch.float16)])
@pytest.mark.parametrize("chunk,n_one", [(70, 60), (1, 41), (250, 100), (3, 9)])
def test_paged_attention_single_tokens_beside_a_chunk(hq, hkv, d, dtype, chunk, n_one):
    """A serving step: decode rows and one prompt chunk in one call, at context
    lengths that are split and not."""
    r = random.Random(chunk)
    new = [1] * n_one
    new[n_one // 3] = chunk
    new[n_one // 2] = 0
    new[-1] = 2
    ctx = [r.choice([0, 5, 63, 700, 2500]) for _ in new]
    q, kc, vc, tables, lens, ids = paged_case(new, ctx, hq, hkv, d, dtype, 32, chunk, n_one + 2)
    ref = paged_reference(q, kc, vc, tables, lens, new, ids, d ** -0.5)
    for most in (max(lens), 40000):
        wide = tables
        if most > max(lens):
            wide = torch.cat([tables, tables[:, :1].expand(-1, most // 32)], 1).contiguous()
        err = i32([0])
        out = run_paged(q, kc, vc, wide, lens, new, ids, err=err, max_kv=most)
        assert int(err) == 0
        check_attention(out, *ref, max(lens), d, dtype)


@pytest.mark.parametrize("group", [1, 5, 8, 9, 16, 17, 32, 33, 100, 128])
@pytest.mark.parametrize("single", [False, True])
def test_paged_attention_head_groups(group, single):
    new = [1] * 3 if single else [4, 1, 0, 37]
    ctx = [130, 0, 2050] if single else [130, 0, 4, 2050]
    q, kc, vc, tables, lens, ids = paged_case(new, ctx, group * 2, 2, 128, torch.bfloat16, 64, group)
    out = run_paged(q, kc, vc, tables, lens, new, ids, single=single)
    ref = paged_reference(q, kc, vc, tables, lens, new, ids, 128 ** -0.5)
    check_attention(out, *ref, max(lens), 128, torch.bfloat16)


@pytest.mark.parametrize("group", [7, 33, 128])
def test_packed_attention_head_groups(group):
    lens = [1, 0, 50, 300]
    q, k, v = rows(sum(lens), group, 1, 64, torch.float16, group)
    out = run_packed(q, k, v, lens)
    check_attention(out, *packed_reference(q, k, v, lens, None, 64 ** -0.5), 300, 64, torch.float16)


@pytest.mark.parametrize("single", [False, True])
@pytest.mark.parametrize("page", [128, 512])
def test_paged_attention_flags_a_bad_large_page(single, page):
    new = [1, 1] if single else [9, 200]
    q, kc, vc, tables, lens, ids = paged_case(new, [1500, 1900], 4, 1, 128, torch.bfloat16, page, 6, junk=0.0)
    gone = tables[ids[1], 2].long()
    k2, v2 = kc.clone(), vc.clone()
    k2[gone], v2[gone] = 0, 0
    ref = paged_reference(q, k2, v2, tables, lens, new, ids, 128 ** -0.5)
    for bad in (-1, kc.shape[0], -(1 << 31)):
        t2, err = tables.clone(), i32([0])
        t2[ids[1], 2] = bad
        out = run_paged(q, kc, vc, t2, lens, new, ids, err=err, single=single)
        assert int(err) & 1
        check_attention(out, *ref, max(lens), 128, torch.bfloat16)


def offset_by(t, n):
    """t's values in memory that starts n elements into an allocation."""
    flat = torch.empty(t.numel() + n, dtype=t.dtype, device=DEV)[n:]
    return flat.view(t.shape).copy_(t)


def test_attention_on_rows_that_are_16_byte_aligned_only():
    hq, hkv, d, dtype = 6, 2, 64, torch.bfloat16
    lens = [33, 200, 1]
    q, k, v = rows(sum(lens), hq, hkv, d, dtype, 3, False)
    q, k, v, out = (offset_by(t, 8) for t in (q, k, v, q))
    run_packed(q, k, v, lens, out=out)
    check_attention(out, *packed_reference(q, k, v, lens, None, d ** -0.5), 200, d, dtype)
    for new, single in (([5, 60], False), ([1, 1], True)):
        q, kc, vc, tables, full, ids = paged_case(new, [300, 40], hq, hkv, d, dtype, 16, 8)
        q, kc, vc, out = (offset_by(t, 8) for t in (q, kc, vc, q))
        run_paged(q, kc, vc, tables, full, new, ids, out=out, single=single)
        ref = paged_reference(q, kc, vc, tables, full, new, ids, d ** -0.5)
        check_attention(out, *ref, max(full), d, dtype)
    with pytest.raises(RuntimeError, match="aligned"):
        run_packed(offset_by(q, 4)[:2], offset_by(kc[0].transpose(0, 1)[:2].contiguous(), 8),
                   offset_by(vc[0].transpose(0, 1)[:2].contiguous(), 8), [2])


def test_attention_on_two_streams_at_once():
    """Calls that overlap, each with a workspace of its own."""
    cases = [paged_case([1] * 3, [20000, 9000, 50], 8, 1, 128, torch.bfloat16, 64, s) for s in (1, 2)]
    refs = [paged_reference(c[0], c[1], c[2], c[3], c[4], [1] * 3, c[5], 128 ** -0.5) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    outs = [[torch.empty_like(c[0]) for _ in range(6)] for c in cases]
    args = [(c[0], c[1], c[2], c[3], i32(c[4]), None, i32(c[5])) for c in cases]
    torch.cuda.synchronize()
    for j in range(6):
        for s, a, o, c in zip(streams, args, outs, cases):
            with torch.cuda.stream(s):
                _native.ops().paged_attention(*a, o[j], max(c[4]), 128 ** -0.5, None)
    torch.cuda.synchronize()
    for o, ref, c in zip(outs, refs, cases):
        for x in o:
            check_attention(x, *ref, max(c[4]), 128, torch.bfloat16)
            assert torch.equal(x, o[0])


def test_two_captured_calls_in_one_pool():
    """Two graphs that share a memory pool, replayed in turn: neither reads what
    the other left in a workspace."""
    cases = [paged_case([1] * 2, [12000, 300], 8, 2, 128, torch.float16, 64, 4),
             paged_case([40, 2], [6000, 9000], 8, 2, 128, torch.float16, 64, 5)]
    graphs, outs, refs, pool = [], [], [], None
    for j, c in enumerate(cases):
        new = [1] * 2 if j == 0 else [40, 2]
        a = (c[0], c[1], c[2], c[3], i32(c[4]), None if j == 0 else i32(starts(new)), i32(c[5]))
        refs.append(paged_reference(c[0], c[1], c[2], c[3], c[4], new, c[5], 128 ** -0.5))
        out = torch.zeros_like(c[0])
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, pool=pool):
            _native.ops().paged_attention(*a, out, max(c[4]), 128 ** -0.5, None)
        pool = g.pool()
        graphs.append((g, a))
        outs.append(out)
    for turn in ((0, 1), (1, 0), (0, 0, 1, 1)):
        for o in outs:
            o.zero_()
        for j in turn:
            graphs[j][0].replay()
        torch.cuda.synchronize()
        for o, ref, c in zip(outs, refs, cases):
            check_attention(o, *ref, max(c[4]), 128, torch.float16)


def test_page_tables_grid_of_slots_with_ends_and_refusals():
    """More than 1024 slots (a second kernel writes them), requests that end,
    one that finds no pages, and requests without new tokens between."""
    page, width, n_pages = 16, 60, 200
    ctx = [100, 0, 37, 960, 16, 0, 5]
    new = [700, 0, 1, 1, 500, 1500, 0]
    done = [1, 0, 0, 0, 1, 0, 1]
    free = list(range(n_pages))
    random.Random(3).shuffle(free)
    tables, held = [], 0
    for c in ctx:
        n = -(-c // page)
        tables.append(free[held:held + n] + [-1] * (width - n))
        held += n
    free = free[held:] + [0] * held
    cap = sum(new) + 37
    got, err = run_tables(ctx, new, done, free, n_pages - held, tables, page, cap)
    want = page_tables_reference(ctx, new, done, free, n_pages - held, tables, page, cap)
    assert err == 8
    for key in want:
        assert got[key] == want[key], key
    assert want["kv"][3] == 960 and want["kv"][5] == 0 and want["kv"][0] == 700


def test_bad_arguments_leave_the_stream_usable():
    """A refused call launches nothing and the next one runs."""
    q, k, v = rows(8, 4, 2, 64, torch.bfloat16, 1)
    for call in (lambda: _native.ops().packed_attention(q, k, v, i32([0, 8]), None, torch.empty_like(q), 0.0, None),
                 lambda: _native.ops().packed_attention(q[:, :3], k, v, i32([0, 8]), None,
                                                        torch.empty_like(q[:, :3]), 1.0, None)):
        with pytest.raises(RuntimeError):
            call()
    out = run_packed(q, k, v, [8])
    check_attention(out, *packed_reference(q, k, v, [8], None, 0.125), 8, 64, torch.bfloat16)


def test_rows_that_overlap_are_refused():
    """An expanded tensor's rows lie in one place (stride 0)."""
    q, k, v = rows(8, 4, 2, 64, torch.bfloat16, 1, False)
    same = {n: t[:1].expand(8, -1, -1) for n, t in (("q", q), ("k", k), ("v", v))}
    out, cu = torch.zeros_like(q), i32([0, 8])
    for a in ((same["q"], k, v), (q, same["k"], same["v"])):
        with pytest.raises(RuntimeError, match="overlap"):
            _native.ops().packed_attention(*a, cu, None, out, 0.125, None)
    kc = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16, device=DEV)
    slots = torch.arange(8, device=DEV)
    with pytest.raises(RuntimeError, match="overlap"):
        _native.ops().paged_append(same["k"], same["v"], slots, None, None, kc, kc.clone(), None)
    with pytest.raises(RuntimeError, match="overlap"):
        _native.ops().paged_attention(same["q"], kc, kc, i32([[0]] * 8), i32([1] * 8), None, None, out,
                                      16, 0.125, None)
    assert not out.any() and not kc.any()


@pytest.mark.parametrize("group,hkv,d", [(2, 3, 128), (32, 2, 64), (64, 1, 128), (96, 2, 64), (16, 1, 128)])
def test_packed_attention_whole_tiles(group, hkv, d):
    """Sequences that fill tiles (their outputs leave as boxes) and do not."""
    lens = [128, 200, 1, 64]
    q, k, v = rows(sum(lens), group * hkv, hkv, d, torch.bfloat16, group)
    out = torch.full_like(q.contiguous(), 7.0)
    tail = torch.full((3, *out.shape[1:]), 7.0, dtype=out.dtype, device=DEV)
    out = torch.cat([out, tail])
    _native.ops().packed_attention(torch.cat([q, q[:3]]), torch.cat([k, k[:3]]), torch.cat([v, v[:3]]),
                                   i32(starts(lens)), None, out, d ** -0.5, None)
    check_attention(out[:-3], *packed_reference(q, k, v, lens, None, d ** -0.5), 200, d, torch.bfloat16)
    assert bool((out[-3:] == 7).all())
