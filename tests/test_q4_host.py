"""The 4-bit cache without a GPU: its entry points reject bad arguments before any
device call, and the format's restatement keeps its promises."""
import pytest
import torch

from tests import q4_helpers as Q
from tide_b200 import _native, capi

P = 1 << 20  # an aligned address that no call below follows
BAD, NOT_HERE, ALIGN = capi.ERR_INVALID, capi.ERR_UNSUPPORTED, capi.ERR_ALIGNMENT


def append(**kw):
    a = dict(dtype=capi.DTYPE_BF16, q=P, qs=0, k=P, v=P, stride=0, qw=None, kw=None, eps=1e-6, freq=P,
             scaling=1.0, pos=P, slots=P, n_map=8, ids=None, live=None, n=8, hq=8, hkv=2, d=128,
             q_out=P, cache=P, n_pages=4, page=16, err=None)
    a.update(kw)
    return _native.lib().tide_paged_append_q4(*a.values(), None)


def read(**kw):
    a = dict(dtype=capi.DTYPE_F16, cache=P, n_pages=4, page=16, slots=P, n=8, hkv=2, d=64, k=P, v=P,
             err=None)
    a.update(kw)
    return _native.lib().tide_paged_read_q4(*a.values(), None)


def attend(**kw):
    a = dict(dtype=capi.DTYPE_BF16, q=P, qs=0, cache=P, n_pages=16, page=16, tables=P, width=8,
             n_req=4, lens=P, cu=P, ids=None, n_seqs=2, live=None, out=P, n=8, hq=8, hkv=2, d=128,
             max_kv=100, scale=0.1, ws=P, ws_bytes=1 << 40, err=None)
    a.update(kw)
    return _native.lib().tide_paged_attention_q4(*a.values(), None)


@pytest.mark.parametrize("kw,rc", [
    (dict(dtype=capi.DTYPE_F32), NOT_HERE), (dict(d=96), NOT_HERE), (dict(page=24), BAD),
    (dict(page=0), BAD), (dict(n_pages=0), BAD), (dict(n_pages=1 << 31), BAD), (dict(hkv=0), BAD),
    (dict(n=-1), BAD), (dict(n_map=7), BAD), (dict(n_map=-1, ids=P), BAD), (dict(hq=0), BAD),
    (dict(qs=8 * 128 - 8), BAD), (dict(qs=8 * 128 + 4), BAD), (dict(stride=2 * 128 - 8), BAD),
    (dict(stride=2 * 128 + 2), BAD), (dict(v=None), BAD), (dict(k=None), BAD),
    (dict(k=None, v=None), BAD), (dict(q_out=None), BAD), (dict(pos=None), BAD), (dict(slots=None), BAD),
    (dict(cache=None), BAD), (dict(cache=P + 8), ALIGN), (dict(q=P + 2), ALIGN), (dict(k=P + 8), ALIGN),
    (dict(q_out=P + 4), ALIGN)])
def test_append_refusals(kw, rc):
    assert append(**kw) == rc
    assert _native.lib().tide_last_error()


@pytest.mark.parametrize("kw,rc", [
    (dict(dtype=capi.DTYPE_F32), NOT_HERE), (dict(d=80), NOT_HERE), (dict(page=8), BAD),
    (dict(n_pages=0), BAD), (dict(n=-1), BAD), (dict(hkv=0), BAD), (dict(slots=None), BAD),
    (dict(k=None), BAD), (dict(v=P + 8), ALIGN), (dict(cache=P + 2), ALIGN)])
def test_read_refusals(kw, rc):
    assert read(**kw) == rc
    assert _native.lib().tide_last_error()


@pytest.mark.parametrize("kw,rc", [
    (dict(dtype=capi.DTYPE_F32), NOT_HERE), (dict(d=256), NOT_HERE), (dict(hq=9), BAD),
    (dict(hq=258), BAD), (dict(hkv=0), BAD), (dict(page=48), NOT_HERE), (dict(page=8), NOT_HERE),
    (dict(max_kv=129), BAD), (dict(max_kv=-1), BAD), (dict(n_pages=0), NOT_HERE),
    (dict(scale=0.0), BAD), (dict(scale=float("nan")), BAD), (dict(scale=float("inf")), BAD),
    (dict(cu=None), BAD), (dict(n_seqs=5), BAD), (dict(n=-1), BAD), (dict(tables=None), BAD),
    (dict(lens=None), BAD), (dict(out=None), BAD), (dict(cache=P + 8), ALIGN), (dict(q=P + 8), ALIGN),
    (dict(qs=1020), BAD), (dict(ws=None), capi.ERR_WORKSPACE), (dict(ws_bytes=16), capi.ERR_WORKSPACE),
    (dict(ws=P + 4), capi.ERR_WORKSPACE)])
def test_attention_refusals(kw, rc):
    kw = dict(dict(n=1000, max_kv=100), **kw)
    assert attend(**kw) == rc
    assert _native.lib().tide_last_error()


def test_empty_calls_do_nothing():
    assert append(n=0, q=None, k=None, v=None, slots=None) == capi.OK
    assert read(n=0, cache=None) == capi.OK
    assert attend(n=0, q=None) == capi.OK
    assert attend(n_seqs=0, q=None) == capi.OK


def test_operators_are_registered_and_have_no_cpu_kernel():
    ops = _native.ops()
    cache = torch.zeros(2, 1, 1, 18 * 64, dtype=torch.uint8)
    k = torch.zeros(3, 1, 64, dtype=torch.float16)
    slots = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(NotImplementedError):
        ops.paged_read_q4(cache, slots, k, k.clone(), None)
    for name in ("paged_append_q4", "paged_attention_q4"):
        assert hasattr(ops, name), name


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_values_are_near_and_of_the_rows_type(dtype):
    """Within half a step of what was put in, exactly a number of the rows' type,
    zero staying zero, for groups of one sign, of two, and of tiny numbers."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(40, 128, generator=g) * torch.logspace(-6, 3, 40)[:, None]
    x[::3] = x[::3].abs()
    x[1::5, 32:64] = 0
    x = x.to(dtype)
    c, z, s = Q.quantise(x, dtype)
    v = Q.values(x, dtype)
    assert torch.equal(v, v.to(dtype).double())
    assert bool(((v - x.double()).abs().unflatten(-1, (-1, 32)) <= s[..., None] / 2).all())
    assert bool((v[x == 0] == 0).all())
    assert int(c.min()) >= 0 and int(c.max()) <= 15 and int(z.min()) >= 0 and int(z.max()) <= 15


@pytest.mark.parametrize("d", [64, 128])
def test_packing_is_the_documented_layout(d):
    g = torch.Generator().manual_seed(4)
    k, v = (torch.randn(2, 3, 32, d, generator=g).to(torch.bfloat16) for _ in range(2))
    cache = Q.pack(k, v, torch.bfloat16)
    assert cache.shape == (2, 3, 2, 18 * d)
    for page, head, token in ((0, 0, 0), (1, 2, 31), (1, 0, 18), (0, 1, 7)):
        got = Q.token_values(cache, page, head, token, d)
        for x, y in zip((k, v), got):
            assert Q.values(x[page, head, token], torch.bfloat16).tolist() == y


def test_numbers_next_to_the_types_largest_stay_finite():
    x = torch.full((1, 64), 65504.0, dtype=torch.float16)
    x[0, 40] = -65504.0
    assert bool(Q.values(x, torch.float16).half().isfinite().all())
    y = torch.full((1, 64), torch.finfo(torch.bfloat16).max, dtype=torch.bfloat16)
    y[0, 3] = -y[0, 3]
    assert bool(Q.values(y, torch.bfloat16).to(torch.bfloat16).isfinite().all())


def test_the_paged_cache_and_generate_refuse_what_4_bits_cannot():
    from tests.test_mask_refusals_host import Reached, generate
    from tide_b200.paged import PagedKVCache

    cpu = torch.device("cpu")
    for bits, d, dtype in ((8, 128, torch.bfloat16), (4, 96, torch.bfloat16), (4, 128, torch.float32)):
        with pytest.raises(ValueError):
            PagedKVCache(1, 2, 4, 16, 2, d, 64, dtype, cpu, bits=bits)
    c = PagedKVCache(2, 2, 4, 32, 2, 128, 64, torch.bfloat16, cpu, bits=4)
    assert c.k == [] and [tuple(x.shape) for x in c.kv] == [(4, 2, 2, 2304)] * 2
    for kw in (dict(kv_bits=8, live=True, paged=True), dict(kv_bits=4), dict(kv_bits=4, live=True)):
        with pytest.raises(ValueError, match="kv_bits"):
            generate(**kw)
    with pytest.raises(Reached):
        generate(kv_bits=4, live=True, paged=True)


def test_reading_a_16_bit_cache_flags_slots_outside_it():
    from tide_b200.paged import PagedKVCache

    c = PagedKVCache(2, 2, 3, 16, 2, 64, 64, torch.float32, torch.device("cpu"))
    for side in (c.k, c.v):
        for x in side:
            x.normal_()
    k, v = c.read(1, torch.tensor([17, -1, 47], dtype=torch.int64))
    assert torch.equal(k[0], c.k[1][1, :, 1]) and torch.equal(v[2], c.v[1][2, :, 15]) and not k[1].any()
    assert int(c.error_word) == 0
    k, v = c.read(0, torch.tensor([48, 3, -2, 1 << 60], dtype=torch.int64))
    assert torch.equal(v[1], c.v[0][0, :, 3]) and not k[[0, 2, 3]].any() and not v[[0, 2, 3]].any()
    assert int(c.error_word) == capi.DEVERR_POSITION


@pytest.mark.parametrize("kw", [
    dict(d=0), dict(d=-64), dict(d=96), dict(n=0), dict(n=1 << 62), dict(n_seqs=0), dict(n_seqs=1 << 62),
    dict(n_req=-1), dict(n_req=1 << 62), dict(hq=0), dict(hkv=0), dict(hq=1 << 62), dict(hq=1024), dict(max_kv=-1),
    dict(max_kv=1 << 62)], ids=str)
def test_no_workspace_for_what_the_call_refuses(kw):
    a = dict(n=800, n_seqs=2, n_req=4, hq=8, hkv=2, d=128, max_kv=100)
    assert _native.lib().tide_paged_attention_q4_workspace_size(*a.values()) > 0
    a.update(kw)
    assert _native.lib().tide_paged_attention_q4_workspace_size(*a.values()) == 0


def test_the_workspace_of_the_largest_sizes():
    most = (1 << 30) - 1
    for n, n_seqs in ((most, most), (most, 1), (most, 1 << 20)):
        got = _native.lib().tide_paged_attention_q4_workspace_size(n, n_seqs, 8, 65536, 65536 // 2, 128, most)
        assert got < 1 << 62 and (n == n_seqs or got > 1 << 40)  # (few rows, or one sequence's pages)


def test_no_workspace_for_single_tokens_where_there_are_offsets():
    """More tokens than sequences come with offsets: 4000 tokens a sequence go to the
    tiles alone, whose 16-bit pages for 2 x 1000 keys of a head of 64 are 512 KB."""
    got = _native.lib().tide_paged_attention_q4_workspace_size(8000, 2, 2, 8, 1, 64, 1000)
    assert 1 << 19 <= got < 1 << 20


@pytest.mark.parametrize("held,other", [(torch.bfloat16, torch.float16), (torch.float16, torch.bfloat16)])
def test_the_paged_cache_refuses_rows_of_another_type(held, other):
    from tide_b200.paged import PagedKVCache

    c = PagedKVCache(1, 2, 4, 16, 2, 64, 64, held, torch.device("cpu"), bits=4)
    slots, freq = torch.arange(3), torch.ones(32)
    a, b = torch.zeros(3, 2, 64, dtype=held), torch.zeros(3, 2, 64, dtype=other)
    for k, v in ((b, b), (a, b), (b, a)):
        with pytest.raises(ValueError, match="cache in 4 bits"):
            c.append(0, k, v, slots)
    for q, k, v in ((b, b, b), (b, a, a), (a, b, a), (a, a, b)):
        with pytest.raises(ValueError, match="cache in 4 bits"):
            c.append_rotated(0, q, k, v, slots, slots, freq)
    for chunk in (False, True):
        with pytest.raises(ValueError, match="cache in 4 bits"):
            c.attend(0, b, 0.1, chunk=chunk)
