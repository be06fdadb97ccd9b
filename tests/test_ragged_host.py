"""The entry points of the ragged operators reject bad arguments before any
device call, and their references agree with themselves."""
import pytest
import torch

from tests.ragged_helpers import attention_rows, page_tables_reference
from tide_b200 import _native, capi

P = 1 << 20  # an aligned address that no call below follows


def packed(**kw):
    a = dict(dtype=capi.DTYPE_BF16, q=P, k=P, v=P, qs=0, ks=0, cu=P, n_seqs=2, zeros=None, out=P,
             n=8, hq=8, hkv=2, d=128, scale=0.1, err=None)
    a.update(kw)
    return _native.lib().tide_packed_attention(*a.values(), None)


def paged(**kw):
    a = dict(dtype=capi.DTYPE_BF16, q=P, qs=0, kc=P, vc=P, n_pages=16, page=16, tables=P, width=8,
             n_req=4, lens=P, cu=P, ids=None, n_seqs=2, live=None, out=P, n=8, hq=8, hkv=2, d=128,
             max_kv=100, scale=0.1, ws=None, ws_bytes=0, err=None)
    a.update(kw)
    return _native.lib().tide_paged_attention(*a.values(), None)


def append(**kw):
    a = dict(dtype=capi.DTYPE_BF16, k=P, v=P, stride=0, slots=P, n_map=8, ids=None, live=None, n=8,
             hkv=2, d=128, kc=P, vc=P, n_pages=4, page=16, err=None)
    a.update(kw)
    return _native.lib().tide_paged_append(*a.values(), None)


def tables(**kw):
    a = dict(ctx=P, new=P, done=None, n=4, free=P, n_free=P, n_pages=16, tables=P, width=8, page=16,
             n_free_out=P, kv=P, cu=P, slots=P, pos=P, n_slots=64, err=None)
    a.update(kw)
    return _native.lib().tide_page_tables(*a.values(), None)


BAD, NOT_HERE, ALIGN = capi.ERR_INVALID, capi.ERR_UNSUPPORTED, capi.ERR_ALIGNMENT


@pytest.mark.parametrize("kw,rc", [
    (dict(dtype=capi.DTYPE_F32), NOT_HERE), (dict(d=96), NOT_HERE), (dict(hq=7), BAD),
    (dict(hkv=0), BAD), (dict(hq=258, hkv=2), BAD), (dict(scale=0.0), BAD), (dict(scale=-1.0), BAD),
    (dict(scale=float("nan")), BAD), (dict(scale=float("inf")), BAD), (dict(n=-1), BAD),
    (dict(n_seqs=-1), BAD), (dict(qs=8 * 128 - 8), BAD), (dict(ks=2 * 128 + 4), BAD),
    (dict(q=None), BAD), (dict(cu=None), BAD), (dict(out=P + 8), ALIGN), (dict(k=P + 2), ALIGN)])
def test_packed_attention_refusals(kw, rc):
    assert packed(**kw) == rc
    assert _native.lib().tide_last_error()


@pytest.mark.parametrize("kw,rc", [
    (dict(dtype=capi.DTYPE_F32), NOT_HERE), (dict(d=256), NOT_HERE), (dict(hq=9), BAD),
    (dict(page=24), NOT_HERE), (dict(page=8), NOT_HERE), (dict(max_kv=129), BAD),
    (dict(max_kv=-1), BAD), (dict(n_pages=0), BAD), (dict(scale=0.0), BAD), (dict(cu=None), BAD),
    (dict(n_seqs=5), BAD), (dict(tables=None), BAD), (dict(lens=None), BAD),
    (dict(vc=P + 8), ALIGN), (dict(qs=1020), BAD), (dict(n_pages=1 << 31), BAD)])
def test_paged_attention_refusals(kw, rc):
    assert paged(**kw) == rc
    assert _native.lib().tide_last_error()


@pytest.mark.parametrize("kw,rc", [
    (dict(dtype=capi.DTYPE_F32), NOT_HERE), (dict(d=80), NOT_HERE), (dict(n_map=7), BAD),
    (dict(stride=2 * 128 - 8), BAD), (dict(stride=2 * 128 + 4), BAD), (dict(v=None), BAD),
    (dict(slots=None), BAD), (dict(page=0), BAD), (dict(n_pages=0), BAD), (dict(n=-1), BAD),
    (dict(kc=P + 8), ALIGN), (dict(hkv=0), BAD)])
def test_paged_append_refusals(kw, rc):
    assert append(**kw) == rc
    assert _native.lib().tide_last_error()


@pytest.mark.parametrize("kw", [
    dict(n=0), dict(n=8193), dict(n_pages=0), dict(width=0), dict(page=0), dict(n_slots=-1),
    dict(ctx=None), dict(free=None), dict(slots=None), dict(width=1 << 30), dict(cu=None)])
def test_page_tables_refusals(kw):
    assert tables(**kw) == BAD
    assert _native.lib().tide_last_error()


def test_empty_calls_do_nothing():
    assert packed(n=0, q=None, k=None, v=None, out=None) == capi.OK
    assert packed(n_seqs=0) == capi.OK
    assert paged(n=0, q=None) == capi.OK
    assert append(n=0, k=None, v=None, slots=None) == capi.OK


def test_operators_are_registered_and_have_no_cpu_kernel():
    ops = _native.ops()
    q = torch.zeros(4, 2, 128, dtype=torch.bfloat16)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(NotImplementedError):
        ops.packed_attention(q, q, q, cu, None, q.clone(), 0.1, None)
    for name in ("paged_attention", "paged_append", "page_tables"):
        assert hasattr(ops, name), name


def test_reference_zero_keys_are_zero_keys():
    """The reference's zero keys against keys and values that are zero."""
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(5, 2, 16, generator=g) for _ in range(3))
    last = torch.full((5,), 7)
    full_k, full_v = torch.cat([k, torch.zeros(3, 2, 16)]), torch.cat([v, torch.zeros(3, 2, 16)])
    a = attention_rows(q, full_k, full_v, last, None, 0.3)[0]
    b = attention_rows(q, k, v, last, torch.full((5,), 3), 0.3)[0]
    torch.testing.assert_close(a, b)


def test_reference_hands_pages_back_and_out():
    r = page_tables_reference([5, 4, 0], [0, 1, 3], [1, 0, 0], [9, 8, 0, 0, 0], 2,
                              [[1, 2], [3, -1], [-1, -1]], 4, 6)
    assert r["n_free"] == 2 and r["free"][:4] == [9, 8, 1, 2]
    assert r["tables"] == [[1, 2], [3, 2], [1, -1]]
    assert r["kv"] == [0, 5, 3] and r["cu"] == [0, 0, 1, 4]
    assert r["slots"] == [8, 4, 5, 6, -1, -1] and r["pos"] == [4, 0, 1, 2, 0, 0]
