"""Prompts into the paged decoder's cache: tokens of any layout, and errors that
a kernel flags while they are processed."""
import pytest
import torch

from tests.test_gpu_live import _qwen3_hd128
from tests.test_gpu_live_ragged import DEV, engine
from tide_b200.paged import PagedLiveDecoder

pytestmark = pytest.mark.gpu


def test_extend_takes_tokens_of_any_layout(tmp_path):
    """A slice of a [requests, tokens] array, whose rows do not lie side by side."""
    model = _qwen3_hd128()
    ids = torch.randint(0, 512, (2, 24), generator=torch.Generator().manual_seed(3)).to(DEV)
    _, rt = engine(tmp_path, model, ids)
    one, two = (PagedLiveDecoder(rt, 2, 32) for _ in range(2))
    a = one.extend(ids[:, :15].reshape(-1), [15, 15])
    b = two.extend(ids[:, :15], [15, 15])
    assert two.lengths == [15, 15] == two.cache.kv_lens.tolist()
    assert torch.equal(a, b)


def test_extend_raises_what_its_kernels_flag(tmp_path):
    """A block table entry outside the pool reads as zeros and is flagged: the
    call that met it raises, the next one does not."""
    model = _qwen3_hd128()
    ids = torch.randint(0, 512, (2, 24), generator=torch.Generator().manual_seed(5)).to(DEV)
    _, rt = engine(tmp_path, model, ids)
    dec = PagedLiveDecoder(rt, 2, 64, page_size=16)
    dec.extend(ids[0, :20], [20, 0])
    was = dec.cache.block_tables[0, 0].clone()
    dec.cache.block_tables[0, 0] = dec.n_pages + 3
    with pytest.raises(RuntimeError, match="error bits 0x1"):
        dec.extend(ids[1, :7], [7, 0])
    dec.cache.block_tables[0, 0] = was
    assert torch.isfinite(dec.extend(ids[1, :5], [0, 5]).float()).all()
    assert dec.lengths == [27, 5] == dec.cache.kv_lens.tolist()
