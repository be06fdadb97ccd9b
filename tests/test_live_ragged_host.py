"""The ragged live paths without a GPU: how survivors are packed, and what is
refused before any kernel."""
from types import SimpleNamespace

import pytest
import torch

from tests.test_live_layers import tiny_llama
from tide_b200.live import _Packed, family_of, live_forward
from tide_b200.paged import PagedKVCache, PagedLiveDecoder


@pytest.mark.parametrize("seed", range(6))
def test_packing_counts_the_exited_tokens_before_each_row(seed):
    g = torch.Generator().manual_seed(seed)
    B, S = 4, 13
    real = torch.rand(B * S, generator=g) < (1.0 if seed == 0 else 0.7)
    real[S:2 * S] &= seed != 1  # (a row of padding only)
    live = real & (torch.rand(B * S, generator=g) < (0.0 if seed == 2 else 0.5))
    pos = real.nonzero()[:, 0]
    order = torch.zeros(B * S, dtype=torch.int64)
    order[pos] = torch.arange(pos.numel())
    first = _Packed.of(pos, B, S, order, None, None)
    assert first.zero_keys is None
    assert first.cu_seqlens.tolist() == [int(real[:b * S].sum()) for b in range(B + 1)]
    rows = live.nonzero()[:, 0]
    p = _Packed.of(rows, B, S, order, first, None)
    assert p.cu_seqlens.dtype == p.zero_keys.dtype == torch.int32
    assert p.cu_seqlens.tolist() == [int(live[:b * S].sum()) for b in range(B + 1)]
    for j, t in enumerate(rows.tolist()):
        b = t // S
        assert p.zero_keys[j] == int((real & ~live)[b * S:t].sum())


def runtime_of(model):
    return SimpleNamespace(_live_family=lambda: family_of(model), model=model, routers={})


def test_padding_needs_a_16_bit_model_and_a_known_head_dim():
    ids = torch.arange(6).view(2, 3)
    mask = torch.tensor([[1, 1, 1], [0, 1, 1]])
    for model in (tiny_llama(), tiny_llama().to(torch.bfloat16)):  # fp32; head_dim 16
        rt = runtime_of(model)
        with pytest.raises(NotImplementedError, match="padding"):
            live_forward(rt, ids, mask)
        with pytest.raises(NotImplementedError, match="packed"):
            live_forward(rt, ids, None, packed=True)
        with pytest.raises(ValueError, match="batch, seq"):
            live_forward(rt, ids, mask[:, :2])


def test_the_paged_decoder_needs_head_dim_128():
    with pytest.raises(NotImplementedError, match="128"):
        PagedLiveDecoder(runtime_of(tiny_llama().to(torch.bfloat16)), 2, 16)


@pytest.mark.parametrize("n_requests,page_size", [(0, 16), (8193, 16), (2, 8), (2, 48)])
def test_the_paged_cache_refuses_shapes(n_requests, page_size):
    with pytest.raises(ValueError):
        PagedKVCache(1, n_requests, 4, page_size, 2, 128, 64, torch.bfloat16, torch.device("cpu"))


def test_the_paged_cache_starts_with_every_page_free():
    c = PagedKVCache(2, 3, 5, 16, 2, 128, 70, torch.float16, torch.device("cpu"))
    assert c.k[1].shape == (5, 2, 16, 128) and c.v[0].dtype == torch.float16
    assert c.block_tables.shape == (3, 5) and int(c.n_free) == 5
    assert sorted(c.free_pages.tolist()) == [0, 1, 2, 3, 4] and not c.kv_lens.any()
