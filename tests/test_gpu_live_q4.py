"""Live decoding over the paged cache in 4 bits.

With the model's own modules (fused_layers=False) the rows that enter the cache
are the same 16-bit ones whatever the cache, so a decoder on a 16-bit cache whose
rows are first replaced by the values that 4 bits hold has to give the same logits
up to roundings, at the tolerance that test_gpu_live_ragged derives.  With the fused
layers what the cache holds is compared bit by bit, for the layer whose input both
sides know."""
import pytest
import torch

from tests import q4_helpers as Q
from tests.test_gpu_live import _qwen3_hd128
from tests.test_gpu_live_ragged import close, engine, mask_of, steps
from tide_b200.paged import PagedKVCache, PagedLiveDecoder
from tide_b200.scheduler import ExitStats

pytestmark = pytest.mark.gpu
DEV = "cuda"


def prompt(B, S, seed):
    return torch.randint(0, 512, (B, S), generator=torch.Generator().manual_seed(seed)).to(DEV)


class Rounded(PagedKVCache):
    """A 16-bit cache of the values that 4 bits hold."""

    def append(self, layer, k, v, slot_map, row_ids=None, n_rows=None):
        if k is not None:
            k, v = (Q.values(x, x.dtype).to(x.dtype) for x in (k, v))
        super().append(layer, k, v, slot_map, row_ids, n_rows)


@pytest.mark.parametrize("graph", [False, True])
def test_decoder_on_4_bits_is_the_decoder_on_their_values(tmp_path, graph):
    model = _qwen3_hd128()
    lens, n = [40, 1, 17, 31], 6
    ids = prompt(4, 40, 13)
    _, rt = engine(tmp_path, model, ids)
    feed = prompt(n, 4, 2)
    a = PagedLiveDecoder(rt, 4, 64, page_size=16, graph=False, fused_layers=False)
    a.cache.__class__ = Rounded
    b = PagedLiveDecoder(rt, 4, 64, page_size=16, graph=graph, fused_layers=False, kv_bits=4)
    assert b.k == [] and len(b.cache.kv) == len(b.fam.layers) and not b._rotates
    mask = mask_of(lens, 40, "left")
    close(b.prefill(ids, mask), a.prefill(ids, mask))
    ref, sa = steps(a, feed[0], n, feed)
    got, sb = steps(b, feed[0], n, feed)
    same = torch.ones(4, dtype=torch.bool, device=DEV)
    for (lr, er), (lg, eg) in zip(ref, got):
        same &= er == eg
        close(lg[same], lr[same])
    assert int(same.sum()) >= 3 and sa.total_exited > 0
    assert b.lengths == [m + n for m in lens] == b.cache.kv_lens.tolist()


def test_fused_layers_fill_the_cache_with_the_rotated_rows(tmp_path):
    """The first layer's keys and values, from the projection's output by the
    formulas in 64 bits, and its attention's logits within the model's tolerance of
    those with the modules."""
    model = _qwen3_hd128()
    lens = [33, 5, 18]
    ids = prompt(3, 33, 3)
    _, rt = engine(tmp_path, model, ids)
    dec = PagedLiveDecoder(rt, 3, 64, page_size=32, kv_bits=4)
    assert dec._rotates
    mask = mask_of(lens, 33, "right")
    dec.prefill(ids, mask)
    fam, layer = dec.fam, dec.fam.layers[0]
    h = fam.embed_tokens(ids[mask.bool()].view(1, -1))
    q, k, v, qw, kw, eps = dec._projected(0, h, None)
    pos = torch.cat([torch.arange(n, device=DEV) for n in lens])
    page = dec.cache.block_tables[torch.repeat_interleave(torch.arange(3), torch.tensor(lens)).to(DEV), pos // 32]
    slots = page.long() * 32 + pos % 32
    gk, gv = dec.cache.read(0, slots)
    kf = Q.turned(k, pos, fam._inv_freq(), kw, eps)[0].float()
    assert torch.equal(gk.double(), Q.values(kf, k.dtype))
    assert torch.equal(gv.double(), Q.values(v, v.dtype))
    none = torch.full((2,), -1, dtype=torch.int64, device=DEV)
    assert not dec.cache.read(0, none)[0].any()


def test_graph_replays_the_eager_step(tmp_path):
    model = _qwen3_hd128()
    ids = prompt(4, 30, 5)
    _, rt = engine(tmp_path, model, ids)
    mask = mask_of([30, 3, 16, 1], 30, "left")
    feed = prompt(18, 4, 8)
    runs = []
    for graph in (False, True):
        dec = PagedLiveDecoder(rt, 4, 50, page_size=16, graph=graph, kv_bits=4)
        dec.prefill(ids, mask)
        runs.append((steps(dec, feed[0], 18, feed), dec))
    ((r0, s0), d0), ((r1, s1), d1) = runs
    for (la, ea), (lb, eb) in zip(r0, r1):
        assert torch.equal(ea, eb)
        torch.testing.assert_close(la, lb, atol=1e-3, rtol=1e-3)
    assert s0.exits_per_layer == s1.exits_per_layer and s0.total_exited > 0
    assert torch.equal(d0.cache.block_tables, d1.cache.block_tables)


def test_zero_pads_the_layers_after_an_exit(tmp_path):
    model = _qwen3_hd128()
    B, S = 8, 21
    ids = prompt(B, S, 29)
    _, rt = engine(tmp_path, model, ids)
    lens = [21, 16, 15, 1, 20, 7, 8, 9]
    dec = PagedLiveDecoder(rt, B, 32, page_size=16, graph=True, kv_bits=4)
    for c in dec.cache.kv:
        c.fill_(0x31)
    tok = dec.prefill(ids, mask_of(lens, S, "right")).argmax(-1)
    st = ExitStats()
    dec.step(tok, st)
    dec.read_stats(st)
    exits = dec.last_exit_layer.cpu().tolist()
    assert any(e >= 0 for e in exits) and any(e < 0 for e in exits)
    slots = torch.tensor([int(dec.cache.block_tables[r, n // 16]) * 16 + n % 16 for r, n in enumerate(lens)],
                         device=DEV)
    for i in range(len(dec.fam.layers)):
        for x in dec.cache.read(i, slots):
            for r, e in enumerate(exits):
                assert bool((x[r] != 0).any()) == (e < 0 or i <= e), (r, e, i)


def test_requests_come_and_go_and_random_caches(tmp_path):
    model = _qwen3_hd128()
    ids = prompt(3, 40, 31)
    _, rt = engine(tmp_path, model, ids)
    dec = PagedLiveDecoder(rt, 3, 64, n_pages=6, page_size=16, graph=True, kv_bits=4)
    dec.extend(torch.cat([ids[0, :30], ids[1, :20]]), [30, 20, 0])
    with pytest.raises(RuntimeError, match="no pages"):
        dec.extend(ids[2], [0, 0, 40])
    dec.step(ids[0, :2])
    assert dec.extend(ids[:0, 0], [0, 0, 0], [False, True, False]) is None
    dec.extend(ids[2], [0, 0, 40])
    one = PagedLiveDecoder(rt, 1, 64, kv_bits=4)
    one.prefill(ids[2:])
    close(dec.step(ids[0, 1:3], requests=[0, 2])[1], one.step(ids[0, 2:3])[0])
    assert dec.lengths == [32, 0, 41] == dec.cache.kv_lens.tolist()
    big = PagedLiveDecoder(rt, 2, 64, kv_bits=4)
    big.fill_random(50, torch.Generator(device=DEV).manual_seed(1))
    assert big.lengths == [50, 50] == big.cache.kv_lens.tolist()
    k, v = big.cache.read(1, big.cache.block_tables[0, :1].long() * 64 + torch.arange(50, device=DEV))
    # N(0, 1) to half a step of a group's range (some 4.5 of 15 steps)
    assert 0.9 < float(k.float().std()) < 1.1 and 0.9 < float(v.float().std()) < 1.1
    assert torch.isfinite(big.step(ids[:2, 0]).float()).all()


@pytest.mark.parametrize("graph", [False, True])
def test_generate_on_4_bits(tmp_path, graph):
    """Greedy tokens of left-padded prompts are those of each prompt alone, up to
    near ties."""
    model = _qwen3_hd128()
    lens = [12, 5, 9]
    ids = prompt(3, 12, 23)
    _, rt = engine(tmp_path, model, ids)
    out = rt.generate(ids, attention_mask=mask_of(lens, 12, "left"), max_new_tokens=5, temperature=0, live=True,
                      paged=True, kv_bits=4, eos_token_id=-1, live_graph=graph)
    assert out.shape == (3, 17) and torch.equal(out[:, :12], ids)
    for r, n in enumerate(lens):
        one = PagedLiveDecoder(rt, 1, 32, kv_bits=4)
        lg = one.prefill(ids[r:r + 1, 12 - n:])
        for j in range(5):
            t = int(out[r, 12 + j])
            assert float(lg[0].max() - lg[0, t]) <= 5e-2, (r, j)
            lg = one.step(out[r, 12 + j:13 + j])


def test_reading_a_16_bit_cache():
    c = PagedKVCache(1, 2, 4, 16, 2, 128, 32, torch.float16, torch.device(DEV))
    k, v = torch.randn(2, 3, 2, 128, device=DEV).half()
    slots = torch.tensor([5, 40, 17], device=DEV)
    c.append(0, k, v, slots)
    gk, gv = c.read(0, torch.tensor([40, -1, 5], device=DEV))
    assert torch.equal(gk[[0, 2]], k[[1, 0]]) and torch.equal(gv[[0, 2]], v[[1, 0]]) and not gk[1].any()
    with pytest.raises(NotImplementedError):
        c.append_rotated(0, k, k, v, slots, slots, torch.ones(64, device=DEV))
