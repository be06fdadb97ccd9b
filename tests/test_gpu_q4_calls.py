"""Calls of the 4-bit cache's attention in which some of the sequences, or some of
its kernels, have nothing to do: against 64-bit references, with what must not be
touched or flagged."""
import pytest
import torch

from tests.gpu_helpers import ptr, stream
from tests.test_gpu_q4 import attend, check, q4_case
from tests.test_gpu_ragged import i32, starts
from tide_b200 import _native, capi

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16


def test_no_long_sequence_among_the_live_ones():
    """Twelve live sequences of 8 tokens before longer ones that are not live: both
    kernels are launched, the tiles' keys split, and no sequence is theirs.  The
    workspace holds what an earlier call left, large numbers here."""
    hq, hkv, d, dtype, most = 8, 2, 128, BF, 8000
    new = [8] * 12 + [100, 40, 33, 51, 0, 0, 0, 0]
    q, cache, held, tables, lens, ids = q4_case(new, [29 * i for i in range(20)], hq, hkv, d, dtype, 16, 7)
    wide = torch.cat([tables, torch.full((20, most // 16), -1, dtype=torch.int32, device=DEV)], 1).contiguous()
    n, lib = q.shape[0], _native.lib()
    size = lib.tide_paged_attention_q4_workspace_size(n, 20, 20, hq, hkv, d, most)
    cu, kv, who = i32(starts(new)), i32(lens), i32(ids)
    for live, byte in ((12, 0x7F), (12, 0), (0, 0x7F), (12, 0xFF), (13, 0x7F)):
        ws = torch.full((size,), byte, dtype=torch.uint8, device=DEV)
        out, err, n_dev = torch.full_like(q, 7.0), i32([0]), i32([live])
        rc = lib.tide_paged_attention_q4(
            capi.DTYPE_BF16, ptr(q), 0, ptr(cache), cache.shape[0], 16, ptr(wide), wide.shape[1], 20, ptr(kv),
            ptr(cu), ptr(who), 20, ptr(n_dev), ptr(out), n, hq, hkv, d, most, d ** -0.5, ptr(ws), size,
            ptr(err), stream())
        capi.check(lib, rc, "tide_paged_attention_q4")
        at = starts(new)[live]
        assert int(err) == 0, (live, byte)
        assert bool((out[at:] == 7).all()), (live, byte)
        if live:
            check(out[:at], q[:at], held, wide, lens, new[:live], ids[:live])


@pytest.mark.parametrize("new", [[150, 0, 40], [0, 200, 0], [4, 0, 2]], ids=str)
@pytest.mark.parametrize("dtype,d", [(BF, 128), (HF, 64)], ids=str)
def test_sequences_without_new_tokens_are_not_looked_at(new, dtype, d):
    """Their requests' pages may be anything (paged_attention's rule): no error, and
    the others' results as before."""
    hq, hkv = 4, 2
    q, cache, held, tables, lens, ids = q4_case(new, [100, 70, 300], hq, hkv, d, dtype, 16, 11)
    err = i32([0])
    want = attend(q, cache, tables, lens, new, ids, err=err)
    check(want, q, held, tables, lens, new, ids)
    broken = tables.clone()
    for n, r in zip(new, ids):
        if n == 0:
            broken[r] = torch.tensor([-1, 1 << 30, cache.shape[0]] * tables.shape[1])[:tables.shape[1]]
    out = attend(q, cache, broken, lens, new, ids, err=err)
    assert int(err) == 0
    assert torch.equal(out, want)


@pytest.mark.parametrize("named", [True, False])
def test_both_kernels_in_rounds(named):
    """Short and long sequences in one call whose 16-bit pages take a round each,
    with and without named requests and a live count from the device."""
    hq, hkv, d, dtype, B, most = 8, 2, 128, HF, 37, 200000
    new = [1 + i % 5 for i in range(B)]
    new[3], new[20], new[21], new[36] = 90, 0, 70, 110
    q, cache, held, tables, lens, ids = q4_case(new, [11 * i for i in range(B)], hq, hkv, d, dtype, 16, 13)
    wide = torch.cat([tables, torch.full((B, most // 16), -1, dtype=torch.int32, device=DEV)], 1).contiguous()
    if not named:
        wide, lens, ids = wide[ids].contiguous(), [lens[r] for r in ids], list(range(B))
    for live in (None, 36, 21, 3, 0):
        out, err = torch.full_like(q, 7.0), i32([0])
        _native.ops().paged_attention_q4(q, cache, wide, i32(lens), i32(starts(new)), i32(ids) if named else None,
                                         out, most, d ** -0.5, err, None if live is None else i32([live]))
        n = B if live is None else live
        at = starts(new)[n]
        assert int(err) == 0 and bool((out[at:] == 7).all())
        if n:
            check(out[:at], q[:at], held, wide, lens, new[:n], ids[:n])


def test_a_captured_call_takes_other_live_counts():
    """The call of the first test, captured once: replays with and without a long
    sequence among the live ones, which all of its kernels have to notice."""
    hq, hkv, d, dtype, most = 8, 2, 128, BF, 8000
    new = [8] * 12 + [100, 40, 33, 51, 0, 0, 0, 0]
    q, cache, held, tables, lens, ids = q4_case(new, [29 * i for i in range(20)], hq, hkv, d, dtype, 16, 17)
    wide = torch.cat([tables, torch.full((20, most // 16), -1, dtype=torch.int32, device=DEV)], 1).contiguous()
    kv, cu, who, err, n_dev = i32(lens), i32(starts(new)), i32(ids), i32([0]), i32([20])
    out = torch.zeros_like(q)

    def call():
        _native.ops().paged_attention_q4(q, cache, wide, kv, cu, who, out, most, d ** -0.5, err, n_dev)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for live in (12, 16, 3, 14, 0, 20, 12):
        n_dev.fill_(live)
        out.fill_(7.0)
        graph.replay()
        at = starts(new)[live]
        assert int(err) == 0 and bool((out[at:] == 7).all()), live
        if live:
            check(out[:at], q[:at], held, wide, lens, new[:live], ids[:live])
