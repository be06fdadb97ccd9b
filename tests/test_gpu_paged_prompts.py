"""Prompts into the paged decoder's cache: tokens of any layout."""
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
