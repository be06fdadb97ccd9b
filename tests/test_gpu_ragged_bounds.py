"""Paged attention with offsets that are not ascending or leave the rows: the
sequences they spoil are skipped and flagged, their neighbours are served,
whichever kernels a call takes and whether it is split over the keys."""
import pytest
import torch

from tests.ragged_helpers import check_attention, paged_reference
from tests.test_gpu_ragged import i32, paged_case
from tide_b200 import _native

pytestmark = pytest.mark.gpu


def served(q, kc, vc, tables, lens, new, ids, cu, max_kv, fine):
    """Runs the call with offsets cu: the rows of the sequences `fine` are
    right, every other row is as it was, the error word is set."""
    hq, d = q.shape[1:]
    wide = torch.cat([tables, tables[:, :1].expand(-1, -(-max_kv // kc.shape[2]))], 1).contiguous()
    out, err = torch.full_like(q, 7.0), i32([0])
    _native.ops().paged_attention(q, kc, vc, wide, i32(lens), i32(cu), i32(ids), out, max_kv, d ** -0.5, err)
    ref = paged_reference(q, kc, vc, tables, lens, new, ids, d ** -0.5)
    rest = torch.ones(q.shape[0], dtype=torch.bool, device=q.device)
    for i in fine:
        rest[cu[i]:cu[i + 1]] = False
    check_attention(out[~rest], *[x[~rest] for x in ref], max(lens), d, q.dtype)
    assert bool((out[rest] == 7).all())
    assert int(err) & 1


@pytest.mark.parametrize("max_kv", [700, 9000, 40000])
@pytest.mark.parametrize("second", [5000, -5, 101, (1 << 31) - 1], ids=str)
def test_tiles_serve_the_neighbours_of_a_bad_sequence(max_kv, second):
    new = [20, 40, 0, 40]
    case = paged_case(new, [300, 100, 0, 513], 8, 2, 128, torch.bfloat16, 64, 3)
    served(*case[:4], case[4], new, case[5], [0, 20, second, 60, 100], max_kv, [0, 3])


@pytest.mark.parametrize("max_kv", [700, 9000])
def test_rows_behind_the_last_sequence_and_a_start_past_the_first_row(max_kv):
    """Rows before the first offset and behind the last belong to no sequence."""
    new = [20, 40, 40]
    case = paged_case(new, [300, 100, 513], 8, 2, 128, torch.bfloat16, 64, 4)
    q, kc, vc, tables, lens, ids = case
    lens = list(lens)
    out, err = torch.full_like(q, 7.0), i32([0])
    wide = torch.cat([tables, tables[:, :1].expand(-1, -(-max_kv // 64))], 1).contiguous()
    _native.ops().paged_attention(q, kc, vc, wide, i32(lens), i32([20, 60]), i32(ids[1:2]), out, max_kv,
                                  128 ** -0.5, err)
    ref = [x[20:60] for x in paged_reference(q, kc, vc, tables, lens, new, ids, 128 ** -0.5)]
    check_attention(out[20:60], *ref, max(lens), 128, q.dtype)
    assert bool((out[:20] == 7).all()) and bool((out[60:] == 7).all()) and int(err) == 0


@pytest.mark.parametrize("max_kv", [104, 4000])
@pytest.mark.parametrize("cu,fine", [
    ([0, 1, 5000], [0]), ([0, 1, -3], [0]), ([2, 1, 2], [1]), ([-1, 1, 2], [1]), ([0, 1, 3], [0])], ids=str)
def test_few_rows_flag_a_bad_sequence(max_kv, cu, fine):
    """Sequences of which two CTAs take one each, and no other kernel runs."""
    new = [1, 1]
    case = paged_case(new, [100, 60], 16, 1, 128, torch.bfloat16, 16, 5)
    served(*case[:4], case[4], new, case[5], cu, max_kv, fine)
