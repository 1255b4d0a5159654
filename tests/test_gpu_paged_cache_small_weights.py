"""Attention over paged caches where one slot has nearly all the weight and its value is 0, so that the others are the whole output.

A token's first slot often is like that. The weights of the others, 2^-gap of the largest, have to keep their precision: fp16 numbers end at
2^-24 and lose bits below 2^-14. The largest weight is between 2^13 and 2^15 when it goes to the tensor core, so that a weight is
held to 2^-25 of that scale, 2^-38 of the largest, or to its type's precision u (u^2 in two parts); the rest is derived in test_gpu_paged_cache.py.
"""
import pytest
import torch

from owoinfer_b200 import ops
from tests.test_gpu_paged_cache import BF16, F, F16, U, attention_64, cu_of, make_cache, near, rows_of, seen_of

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean_status():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    ops.paged_cache_status(clear=True)
    yield
    torch.cuda.synchronize()


def peaked(n, d, dtype, gap, top):
    """A cache of n slots whose slot `top` outdoes the others by `gap` binades for the queries returned with it; what lies there is 0."""
    cache = make_cache([n], 1, d, 16, dtype)
    cache.v.copy_((64.0 * (0.5 + 0.5 * torch.rand(cache.v.shape, generator=torch.Generator().manual_seed(3)))).to(dtype))
    cache.k.zero_()
    place = cache.block_table[0, top // 16].item(), 0, top % 16
    cache.v[place] = 0.0
    cache.k[place] = 1.0
    q = torch.full((1, 3, d), gap * 0.6931471805599453 / d, dtype=torch.float64).to(dtype).cuda()
    return cache, q


def check(cache, q, n, got, lse, parts):
    k, v = rows_of(cache, cache.k, 0, n), rows_of(cache, cache.v, 0, n)
    want, want_lse, size, _ = attention_64(q, k, v, seen_of(torch.tensor([n - 1], device="cuda"), n, 0, 0), 1.0)
    u = U[q.dtype]
    floor = 2.0 ** -38 * v.double().abs().sum(0).repeat_interleave(q.shape[1], 0) if q.dtype == F16 else 0.0
    # (An output below 2^-14 is rounded to multiples of 2^-24.)
    near(got, want, u * want.abs() + (u ** parts + F) * size + floor + 2.0 ** -25, "out")
    near(lse, want_lse, F * (1 + want_lse.abs()), "lse")


CASES = [(64, 0), (64, 63), (500, 3), (2000, 0), (20000, 11111)]


@pytest.mark.parametrize("dtype,d", [(F16, 64), (F16, 128), (BF16, 64)])
@pytest.mark.parametrize("gap", [12.0, 18.5, 25.4])
@pytest.mark.parametrize("n,top", CASES)
def test_decode_keeps_small_weights(dtype, d, gap, n, top):
    cache, q = peaked(n, d, dtype, gap, top)
    for weights in (None, torch.zeros((1, 1, cache.slots), device="cuda")):
        got, lse = ops.attention_paged_decode(q, cache, 1.0, weights=weights)
        check(cache, q, n, got, lse, 2)
    assert ops.paged_cache_status() == 0


@pytest.mark.parametrize("dtype,d", [(F16, 64), (F16, 128), (BF16, 64)])
@pytest.mark.parametrize("gap", [12.0, 18.5, 25.4])
@pytest.mark.parametrize("n,top", CASES)
def test_prompt_keeps_small_weights(dtype, d, gap, n, top):
    cache, q = peaked(n, d, dtype, gap, top)
    got, lse = ops.attention_paged(q, cache, cu_of([1]), 1, 1.0)
    check(cache, q, n, got, lse, 1)
    assert ops.paged_cache_status() == 0
