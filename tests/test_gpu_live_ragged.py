"""Live early exit on ragged batches: padded prompts through the packed
attention of the active rows, and decoding over the paged cache, against each
sequence by itself.

Logits are compared at 5e-2: at these sizes (unit-normed rows of 256, lm_head
weights of 0.02, so a logit is 0.02 * 16 times a unit row's component) some 36
roundings of 2^-9 rms each along 6 bf16 layers give 36^0.5 * 2^-9 * 0.32 =
4e-3 rms, 2e-2 at the 4.5 sigma of 1e5 logits, twice that between two such
runs; fp16 is below.  A token whose score lies within 1e-2 of the threshold
(that error through the router, whose weights are 0.05 and 0.2 over 256 and 64
wide sums, as in test_gpu_live) may be decided either way; its sequence then
differs from there on."""
import numpy as np
import pytest
import torch

from tests.test_gpu_live import _qwen3_hd128, dense_emulation
from tests.test_gpu_runtime import gpt2, llama, tuned_routers
from tide_b200 import TIDEConfig
from tide_b200.paged import PagedLiveDecoder
from tide_b200.runtime import TIDERuntime
from tide_b200.scheduler import ExitStats

pytestmark = pytest.mark.gpu
DEV = "cuda"


def close(a, b):
    torch.testing.assert_close(a.float(), b.float(), atol=5e-2, rtol=5e-2)


def engine(tmp_path, model, ids, layers=(1, 2), share=0.35, threshold=0.6):
    routers = tuned_routers(tmp_path / "router.pt", model, ids, list(layers), [share] * len(layers),
                            threshold)
    return routers, TIDERuntime(model, tmp_path / "router.pt",
                                config=TIDEConfig(exit_threshold=threshold, min_layers=0))


def mask_of(lens, S, side):
    m = torch.zeros(len(lens), S, dtype=torch.long)
    for r, n in enumerate(lens):
        if n:
            m[r, :n] = 1 if side == "right" else 0
            m[r, S - n:] = 1 if side == "left" else m[r, S - n:]
    return m.to(DEV)


@pytest.mark.parametrize("side", ["right", "left"])
@pytest.mark.parametrize("family", ["llama", "hd128"])
def test_live_padded_rows_are_the_rows_alone(tmp_path, family, side):
    model = llama(layers=6) if family == "llama" else _qwen3_hd128()
    lens = [48, 1, 0, 33, 17]
    S = max(lens)
    ids = torch.randint(0, 512, (len(lens), S), generator=torch.Generator().manual_seed(7)).to(DEV)
    routers, rt = engine(tmp_path, model, ids, layers=(1, 3) if family == "llama" else (1, 2))
    mask = mask_of(lens, S, side)
    with torch.no_grad():
        logits = rt(ids, attention_mask=mask, live=True)
    st, exits = rt.last_stats, rt.last_exit_layer.cpu().numpy()
    assert st.total_tokens == sum(lens) and 0 < st.total_exited
    assert st.total_exited + st.remaining_tokens == sum(lens)
    flips = 0
    for r, n in enumerate(lens):
        at = slice(0, n) if side == "right" else slice(S - n, S)
        pad = mask[r] == 0
        assert torch.equal(logits[r, pad], torch.zeros_like(logits[r, pad]))
        assert (exits[r, pad.cpu().numpy()] == -1).all()
        if n == 0:
            continue
        ref, theirs, scores = dense_emulation(model, rt, ids[r:r + 1, at], routers, 0.6, 0)
        differ = np.nonzero(exits[r, at] != theirs)[0]
        if len(differ):
            i = differ[0]
            first = min(x for x in (exits[r, at][i], theirs[i]) if x >= 0)
            assert abs(scores[first][i] - 0.6) <= 1e-2
            flips += 1
            continue
        close(logits[r, at], ref[0])
    assert flips <= 1


def test_live_with_a_batch_of_padding_only(tmp_path):
    model = llama()
    ids = torch.randint(0, 512, (2, 20), generator=torch.Generator().manual_seed(3)).to(DEV)
    _, rt = engine(tmp_path, model, ids)
    logits = rt(ids, attention_mask=torch.zeros_like(ids), live=True)
    assert not logits.any() and rt.last_stats.total_tokens == 0


@pytest.mark.parametrize("family", ["llama", "gpt2", "hd128"])
def test_live_packed_is_the_live_forward(tmp_path, family):
    """Survivors packed, the exited tokens' zero keys counted, against the same
    zeros in the whole layout."""
    model = {"llama": llama, "gpt2": gpt2, "hd128": _qwen3_hd128}[family]()
    ids = torch.randint(0, 512, (4, 60), generator=torch.Generator().manual_seed(9)).to(DEV)
    _, rt = engine(tmp_path, model, ids)
    with torch.no_grad():
        ref = rt(ids, live=True)
        theirs = rt.last_exit_layer
        ours = rt(ids, live=True, packed=True)
    same = (theirs == rt.last_exit_layer).all(1)
    assert rt.last_stats.total_exited > 0 and int(same.sum()) >= 3
    close(ours[same], ref[same])


def steps(dec, tokens, n, feed=None, requests=None):
    """n decode steps: (logits, exit layers) of each; feed: the tokens to take,
    else the greedy ones."""
    out, st = [], ExitStats()
    for j in range(n):
        kw = {} if requests is None else {"requests": requests}
        lg = dec.step(tokens, st, **kw).float().clone()
        out.append((lg, dec.last_exit_layer.clone()))
        tokens = feed[j] if feed is not None else lg.argmax(-1)
    dec.read_stats(st)
    assert st.total_exited + st.remaining_tokens == st.total_tokens == n * tokens.shape[0]
    return out, st


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("fused", [False, True])
def test_paged_decoder_is_the_live_decoder(tmp_path, graph, fused):
    from tide_b200.live import LiveDecoder

    model = _qwen3_hd128()
    B, S, n = 5, 15, 5  # (the third step's positions begin a second page)
    ids = torch.randint(0, 512, (B, S), generator=torch.Generator().manual_seed(29)).to(DEV)
    _, rt = engine(tmp_path, model, ids)
    a = LiveDecoder(rt, B, S + n, graph=False, fused_layers=fused)
    b = PagedLiveDecoder(rt, B, S + n, page_size=16, graph=graph, fused_layers=fused)
    with torch.no_grad():
        first, ours = a.prefill(ids), b.prefill(ids)
    close(ours, first)
    feed = torch.randint(0, 512, (n, B), generator=torch.Generator().manual_seed(1)).to(DEV)
    ref, sa = steps(a, first.argmax(-1), n, feed)
    got, sb = steps(b, first.argmax(-1), n, feed)
    same = torch.ones(B, dtype=torch.bool, device=DEV)
    for (lr, er), (lg, eg) in zip(ref, got):
        same &= er == eg
        close(lg[same], lr[same])
    assert int(same.sum()) >= B - 1 and sa.total_exited > 0
    assert b.lengths == [S + n] * B and b.length == S + n
    assert b.cache.kv_lens.tolist() == b.lengths
    with pytest.raises(RuntimeError, match="full"):
        b.step(feed[0])


def test_paged_decoder_graph_replays_the_eager_step(tmp_path):
    model = _qwen3_hd128()
    B, S = 4, 30
    ids = torch.randint(0, 512, (B, S), generator=torch.Generator().manual_seed(5)).to(DEV)
    _, rt = engine(tmp_path, model, ids)
    mask = mask_of([30, 3, 16, 1], S, "left")
    runs = []
    for graph in (False, True):
        dec = PagedLiveDecoder(rt, B, S + 20, page_size=16, graph=graph)
        first = dec.prefill(ids, mask).argmax(-1)
        runs.append((steps(dec, first, 18), dec))
    ((r0, s0), d0), ((r1, s1), d1) = runs
    for (la, ea), (lb, eb) in zip(r0, r1):
        assert torch.equal(ea, eb)
        torch.testing.assert_close(la, lb, atol=1e-3, rtol=1e-3)
    assert s0.exits_per_layer == s1.exits_per_layer
    assert torch.equal(d0.cache.block_tables, d1.cache.block_tables)
    assert torch.equal(d0.cache.n_free, d1.cache.n_free)


def test_paged_decoder_ragged_requests_are_the_requests_alone(tmp_path):
    """Prompts of several lengths in one cache, one of them in two chunks,
    against a decoder of one request each."""
    model = _qwen3_hd128()
    lens, n = [40, 1, 17, 31], 4
    S = max(lens)
    ids = torch.randint(0, 512, (4, S), generator=torch.Generator().manual_seed(13)).to(DEV)
    _, rt = engine(tmp_path, model, ids)
    feed = torch.randint(0, 512, (n, 4), generator=torch.Generator().manual_seed(2)).to(DEV)
    dec = PagedLiveDecoder(rt, 4, 64, page_size=16, graph=True)
    prompts = [ids[r, :m] for r, m in enumerate(lens)]
    part = dec.extend(torch.cat([prompts[0][:25], prompts[2]]), [25, 0, 17, 0], [True] * 4)
    assert not part[1].any() and not part[3].any()
    rest = dec.extend(torch.cat([prompts[0][25:], prompts[1], prompts[3]]), [15, 1, 0, 31])
    first = torch.where(torch.tensor([[False], [False], [True], [False]], device=DEV), part, rest)
    got, _ = steps(dec, feed[0], n, feed)
    assert dec.lengths == [m + n for m in lens] == dec.cache.kv_lens.tolist()
    flips = 0
    for r in range(4):
        one = PagedLiveDecoder(rt, 1, 64, page_size=32)
        close(first[r], one.prefill(prompts[r][None])[0])
        ref, _ = steps(one, feed[0, r:r + 1], n, feed[:, r:r + 1])
        for (lg, eg), (lr, er) in zip(got, ref):
            if eg[r] != er[0]:
                flips += 1
                break
            close(lg[r], lr[0])
    assert flips <= 1


def test_paged_decoder_zero_pads_the_layers_after_an_exit(tmp_path):
    model = _qwen3_hd128()
    B, S = 8, 21
    ids = torch.randint(0, 512, (B, S), generator=torch.Generator().manual_seed(29)).to(DEV)
    _, rt = engine(tmp_path, model, ids)
    lens = [21, 16, 15, 1, 20, 7, 8, 9]
    dec = PagedLiveDecoder(rt, B, 32, page_size=16, graph=True)
    for c in dec.k + dec.v:
        c.fill_(1.0)
    tok = dec.prefill(ids, mask_of(lens, S, "right")).argmax(-1)
    st = ExitStats()
    dec.step(tok, st)
    dec.read_stats(st)
    exits = dec.last_exit_layer.cpu().tolist()
    assert any(e >= 0 for e in exits) and any(e < 0 for e in exits)
    for r, e in enumerate(exits):
        page = int(dec.cache.block_tables[r, lens[r] // 16])
        for i in range(len(dec.k)):
            for c in (dec.k[i], dec.v[i]):
                row = c[page, :, lens[r] % 16]
                assert bool((row != 0).any()) == (e < 0 or i <= e), (r, e, i)


def test_paged_decoder_requests_come_and_go(tmp_path):
    """A pool too small for all requests at once: one ends, its pages go to
    another, a step runs on some of the requests; the others' tokens are what
    they are without any of this."""
    model = _qwen3_hd128()
    ids = torch.randint(0, 512, (3, 40), generator=torch.Generator().manual_seed(31)).to(DEV)
    _, rt = engine(tmp_path, model, ids)
    feed = torch.randint(0, 512, (6, 3), generator=torch.Generator().manual_seed(4)).to(DEV)
    dec = PagedLiveDecoder(rt, 3, 64, n_pages=6, page_size=16, graph=True)
    dec.extend(torch.cat([ids[0, :30], ids[1, :20]]), [30, 20, 0])
    with pytest.raises(RuntimeError, match="no pages"):
        dec.extend(ids[2], [0, 0, 40])
    got = [steps(dec, feed[0, :2], 2, feed[:, :2])[0]]
    # request 1 gives its two pages back; request 2 takes three
    assert dec.extend(ids[:0, 0], [0, 0, 0], [False, True, False]) is None
    assert int(dec.cache.n_free) == 6 - 2
    dec.extend(ids[2], [0, 0, 40])
    got.append(steps(dec, feed[2, [0, 2]], 3, feed[3:, [0, 2]], requests=[0, 2])[0])
    got.append(steps(dec, feed[5, 2:], 1, feed[5:, 2:], requests=[2])[0])
    with pytest.raises(ValueError, match="ascending"):
        dec.step(feed[0, :2], requests=[2, 0])
    with pytest.raises(ValueError, match="ascending"):
        dec.step(feed[0, :1], requests=[3])
    assert dec.lengths == [35, 0, 44] == dec.cache.kv_lens.tolist()
    one = PagedLiveDecoder(rt, 1, 64)
    one.prefill(ids[:1, :30])
    a = steps(one, feed[0, :1], 2, feed[:, :1])[0] + steps(one, feed[2, :1], 3, feed[3:, :1])[0]
    one.prefill(ids[2:])
    b = steps(one, feed[2, 2:], 3, feed[3:, 2:])[0] + steps(one, feed[5, 2:], 1, feed[5:, 2:])[0]
    seen = [[(lg[0], e[0]) for lg, e in got[0] + got[1]],
            [(lg[-1], e[-1]) for lg, e in got[1] + got[2]]]
    flips = 0
    for ours, ref in zip(seen, (a, b)):
        assert len(ours) == len(ref)
        for (lg, eg), (lr, er) in zip(ours, ref):
            if eg != er[0]:
                flips += 1
                break
            close(lg, lr[0])
    assert flips <= 1


@pytest.mark.parametrize("graph", [False, True])
def test_generate_paged(tmp_path, graph):
    """Greedy tokens of left-padded prompts are those of each prompt alone, up
    to near ties (5e-2, as above) of two tokens."""
    model = _qwen3_hd128()
    lens = [12, 5, 9]
    ids = torch.randint(0, 512, (3, 12), generator=torch.Generator().manual_seed(23)).to(DEV)
    _, rt = engine(tmp_path, model, ids)
    kw = dict(max_new_tokens=5, temperature=0, live=True, paged=True, eos_token_id=-1,
              live_graph=graph)
    out = rt.generate(ids, attention_mask=mask_of(lens, 12, "left"), **kw)
    assert out.shape == (3, 17) and torch.equal(out[:, :12], ids)
    st = rt.last_stats
    assert st.total_tokens == 15 == st.total_exited + st.remaining_tokens
    for r, n in enumerate(lens):
        one = PagedLiveDecoder(rt, 1, 32)
        lg = one.prefill(ids[r:r + 1, 12 - n:])
        for j in range(5):
            t = int(out[r, 12 + j])
            assert float(lg[0].max() - lg[0, t]) <= 5e-2, (r, j)
            lg = one.step(out[r, 12 + j:13 + j])


def test_paged_decoder_refuses_what_it_cannot_take(tmp_path):
    model = _qwen3_hd128()
    ids = torch.randint(0, 512, (2, 8), generator=torch.Generator().manual_seed(3)).to(DEV)
    _, rt = engine(tmp_path, model, ids)
    dec = PagedLiveDecoder(rt, 2, 16)
    with pytest.raises(ValueError, match="new_lens"):
        dec.extend(ids[0], [8])
    with pytest.raises(ValueError, match="new_lens"):
        dec.extend(ids[0], [4, 5])
    with pytest.raises(RuntimeError, match="full"):
        dec.extend(torch.cat([ids[0]] * 3), [24, 0])
    with pytest.raises(ValueError, match="prompt"):
        dec.prefill(ids, mask_of([8, 0], 8, "right"))
    with pytest.raises(ValueError, match="batch, seq"):
        dec.prefill(ids, torch.ones(2, 7, device=DEV))
    with pytest.raises(ValueError, match="requests"):
        dec.step(ids[0][:3], requests=None)
    assert dec.lengths == [0, 0] == dec.cache.kv_lens.tolist()
    dec.fill_random(10, torch.Generator(device=DEV).manual_seed(1))
    assert dec.lengths == [10, 10] == dec.cache.kv_lens.tolist()
    assert torch.isfinite(dec.step(ids[:, 0]).float()).all()
