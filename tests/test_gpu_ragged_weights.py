"""Softmax weights far below the largest one, and at the top of what a kernel
lets them grow to, in the ragged attention operators: one key may hold nearly
all of a row's weight and none of its value, and the rest of the output then
comes from many weights that are small in the rows' 16-bit type."""
import math

import pytest
import torch

from tests.ragged_helpers import attention_rows, check_attention, packed_reference, paged_reference
from tests.test_gpu_ragged import DEV, i32, paged_case, run_packed
from tide_b200 import _native

pytestmark = pytest.mark.gpu
SCALE = math.log(2.0)  # a score is then the exponent of its weight, base 2
DROPS = (21.5, 24.0, 25.25, 26.5)  # of the other keys below the first, per KV head


def check_tail(got, ref, size, reach, n, d, dtype, most):
    """attention_bound's terms, with half a step of the smallest output instead
    of its allowance for subnormals, and for fp16 the weights that are subnormal
    there: a row's largest weight (1 at least of the scaled sum) is 2^7, so
    half a subnormal step, 2^-25, is 2^-32 of it, for n keys of values up to
    `most`."""
    eps = torch.finfo(dtype).eps
    rel = eps / 2 + 2 * (d * 2.0 ** -23 * reach + 2.0 ** -20) + 2 * (n + 2) * 2.0 ** -23
    may = eps / 2 * ref.abs() + rel * size * (1 + eps) + torch.finfo(dtype).smallest_normal * eps / 2
    if dtype == torch.float16:
        may = may + n * 2.0 ** -32 * most
    off = (got.double() - ref).abs()
    assert bool((off <= may).all()), f"off by up to {(off / may).max().item():.3g} of the bound"


def one_large_key(n, hq, hkv, d, dtype, seed, first=0.0):
    """q [n, hq, d], k and v [n, hkv, d]: key 0 of score `first`, with a value
    of 0; the others DROPS below 0, with values of 4 to 8."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    q = torch.zeros(n, hq, d, device=DEV)
    q[:, :, 0] = 1.0
    k = torch.zeros(n, hkv, d, device=DEV)
    k[:, :, 0] = -torch.tensor(DROPS[:hkv], device=DEV)
    k[0, :, 0] = first
    v = 4 + 4 * torch.rand(n, hkv, d, generator=g, device=DEV)
    v[0] = 0
    return q.to(dtype), k.to(dtype), v.to(dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128])
def test_packed_attention_keeps_small_weights(dtype, d):
    n = 2048
    q, k, v = one_large_key(n, 8, 4, d, dtype, d)
    out = run_packed(q, k, v, [n], scale=SCALE)
    check_tail(out, *packed_reference(q, k, v, [n], None, SCALE), n, d, dtype, 8)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("zero", [1, 900])
def test_packed_attention_keeps_small_weights_beside_zero_keys(dtype, zero):
    """Zero keys have score 0: the others are below them."""
    n, d = 1500, 128
    q, k, v = one_large_key(n, 4, 4, d, dtype, zero, first=-DROPS[0])
    zeros = torch.full((n,), zero, dtype=torch.int32, device=DEV)
    out = run_packed(q, k, v, [n], zeros, scale=SCALE)
    check_tail(out, *packed_reference(q, k, v, [n], zeros, SCALE), n, d, dtype, 8)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("new,ctx,single", [
    ([40], [3000], False), ([3, 2], [2000, 900], False), ([1, 1], [3000, 1500], True),
    ([1] * 160, [400] * 160, True)], ids=["chunk", "few", "single", "many"])
def test_paged_attention_keeps_small_weights(dtype, new, ctx, single):
    """The same over the pages, split over the keys or not."""
    hq, hkv, d, page = 8, 4, 128, 32
    q, kc, vc, tables, lens, ids = paged_case(new, ctx, hq, hkv, d, dtype, page, 5)
    q.zero_()
    q[:, :, 0] = 1.0
    for i, r in enumerate(ids):
        _, k, v = one_large_key(lens[r], hq, hkv, d, dtype, i)
        for j in range(0, lens[r], page):
            m, p = min(page, lens[r] - j), int(tables[r, j // page])
            kc[p, :, :m], vc[p, :, :m] = k[j:j + m].transpose(0, 1), v[j:j + m].transpose(0, 1)
    out = torch.empty_like(q)
    cu = i32([sum(new[:i]) for i in range(len(new) + 1)])
    _native.ops().paged_attention(q, kc, vc, tables, i32(lens), None if single else cu, i32(ids), out,
                                  max(lens), SCALE, None)
    ref = paged_reference(q, kc, vc, tables, lens, new, ids, SCALE)
    check_tail(out, *ref, max(lens), d, dtype, 8)


def climbing(n, d, dtype, top, seed):
    """Keys of score 0, and from the second block of keys on of score `top`."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    q = torch.zeros(n, 2, d, device=DEV)
    q[:, :, 0] = 1.0
    k = torch.zeros(n, 1, d, device=DEV)
    k[130:, :, 0] = top
    return q.to(dtype), k.to(dtype), torch.randn(n, 1, d, generator=g, device=DEV).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("top", [6.5, 7.9375, 8.0, 8.0625])
def test_packed_attention_weights_above_the_first_maximum(dtype, top):
    """Scores up to, at and past what a maximum may grow by before the sums
    are rescaled."""
    n, d = 900, 128
    q, k, v = climbing(n, d, dtype, top, 3)
    out = run_packed(q, k, v, [n], scale=SCALE)
    check_attention(out, *packed_reference(q, k, v, [n], None, SCALE), n, d, dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("single", [False, True])
def test_attention_of_huge_scores_is_finite(dtype, single):
    """Scores of 2^24 and a little more: 32 bits hold them to a step of 1 or 2,
    which is a factor of 4 in a weight, but no weight leaves its type's range."""
    n, d, page = 900, 128, 64
    q, k, v = climbing(n, d, dtype, 0.0, 4)
    q[:, :, 0], k[:, :, 0] = 4096.0, 4096.0
    q[:, :, 1], k[130:, :, 1] = 1.0, 7.0
    if single:
        pages = -(-n // page)
        kc = torch.zeros(pages, 1, page, d, dtype=dtype, device=DEV)
        vc = torch.zeros_like(kc)
        kc.view(-1, d)[:n], vc.view(-1, d)[:n] = k[:, 0], v[:, 0]
        out = torch.empty_like(q[:1])
        _native.ops().paged_attention(q[:1].contiguous(), kc, vc, i32([list(range(pages))]), i32([n]), None,
                                      None, out, n, SCALE, None)
    else:
        out = run_packed(q, k, v, [n], scale=SCALE)
    assert bool(out.isfinite().all()) and float(out.abs().max()) <= float(v.abs().max()) * 1.01


def test_the_tail_of_the_reference():
    """The tests' own reference at one case worked out by hand: 1023 keys of
    weight 2^-24 and value 4 beside one of weight 1 and value 0."""
    q = torch.ones(1, 1, 1, dtype=torch.float16, device=DEV)
    k = torch.full((1024, 1, 1), -24.0, dtype=torch.float16, device=DEV)
    v = torch.full((1024, 1, 1), 4.0, dtype=torch.float16, device=DEV)
    k[0], v[0] = 0, 0
    o = attention_rows(q, k, v, torch.tensor([1023], device=DEV), None, SCALE)[0]
    tail = 1023 * 2.0 ** -24
    assert abs(float(o) - 4 * tail / (1 + tail)) <= 1e-12
