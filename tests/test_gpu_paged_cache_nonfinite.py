"""Scores, keys, queries and values that are not finite, on paged key-value caches, against the definitions in 64 bits.

A NaN or an infinity among the scores that a token sees makes its output and its lse NaN (the definition subtracts the largest score); a score
of minus infinity is a weight of 0, and a token all of whose scores are that is one that sees nothing: zeros and minus infinity. The tolerances
of finite values are those of test_gpu_paged_cache.py, where they are derived.
"""
import math

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


def put(cache, pool, b, slot, value, head=slice(None), channel=slice(None)):
    pool[cache.block_table[b, slot // cache.page_size].item(), head, slot % cache.page_size, channel] = value


def expect(cache, b, q, slots, window, sinks, scale):
    """(out, lse, sum p |v|) of the tokens at `slots` of sequence b."""
    end = int(cache.seq_lens[b])
    want, lse, size, _ = attention_64(q, rows_of(cache, cache.k, b, end), rows_of(cache, cache.v, b, end), seen_of(slots, end, window, sinks), scale)
    want[lse == -math.inf] = 0.0
    size[lse == -math.inf] = 0.0
    return want, torch.where(lse == math.inf, math.nan, lse), size


def check(cache, q, new, scale, got, lse, dtype, window=0, sinks=0):
    at = 0
    for b, n in enumerate(new):
        end = int(cache.seq_lens[b])
        want, want_lse, size = expect(cache, b, q[at:at + n], torch.arange(end - n, end, device="cuda"), window, sinks, scale)
        near(got[at:at + n], want, U[dtype] * want.abs() + (U[dtype] + F) * size + 1e-7, "out")
        near(lse[at:at + n], want_lse, F * (1 + want_lse.abs()), "lse")
        at += n


def queries(tokens, heads, d, dtype):
    return torch.randn((tokens, heads, d), generator=torch.Generator().manual_seed(9)).to(dtype).cuda()


# ---------------------------------------------------------------------------------------------------- scores of a prompt

@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 128), (BF16, 64), (F16, 64)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("n,slot", [(1, 0), (40, 0), (40, 1), (40, 5), (130, 129), (200, 16), (256, 128), (300, 0), (300, 260), (700, 300)])
def test_prompt_with_a_key_that_is_not_finite(dtype, d, bad, n, slot):
    """One channel of one key: every row that sees it, in the first pair of key tiles or behind it, and no others."""
    cache = make_cache([n], 2, d, 16, dtype)
    put(cache, cache.k, 0, slot, bad, channel=3)
    q = queries(n, 4, d, dtype)
    got, lse = ops.attention_paged(q, cache, cu_of([n]), n, d ** -0.5)
    check(cache, q, [n], d ** -0.5, got, lse, dtype)
    assert ops.paged_cache_status() == 0


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("n,window,sinks", [(1, 0, 0), (40, 0, 0), (300, 0, 0), (700, 64, 3)])
def test_prompt_with_queries_that_are_not_finite(dtype, d, bad, n, window, sinks):
    cache = make_cache([n], 2, d, 16, dtype)
    q = queries(n, 4, d, dtype)
    for token in {0, 1 % n, 7 % n, n // 2, n - 1}:
        q[token, token % 4, 5] = bad
    got, lse = ops.attention_paged(q, cache, cu_of([n]), n, d ** -0.5, window=window, sinks=sinks)
    check(cache, q, [n], d ** -0.5, got, lse, dtype, window, sinks)


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("slots", [[0], [1], [5], [3900], range(1300, 2600, 128), range(0, 5000, 128)])
def test_prompt_in_parts_with_keys_that_are_not_finite(dtype, d, bad, slots):
    """Few tokens over many slots: parts all of whose tiles have such a score, in a long sequence and in one of a single tile."""
    lens, new = [5000, 100], [3, 2]
    cache = make_cache(lens, 1, d, 32, dtype)
    q = queries(sum(new), 4, d, dtype)
    assert ops.attention_paged_workspace_bytes(cache, sum(new), 4, max(new)) > 256
    for b in range(2):
        for slot in slots:
            if slot < lens[b]:
                put(cache, cache.k, b, slot, bad, channel=slice(0, 2))
    got, lse = ops.attention_paged(q, cache, cu_of(new), max(new), d ** -0.5)
    check(cache, q, new, d ** -0.5, got, lse, dtype)
    q[0, 0, 0] = q[4, 1, 0] = math.nan
    clean = make_cache(lens, 1, d, 32, dtype)
    got, lse = ops.attention_paged(q, clean, cu_of(new), max(new), d ** -0.5)
    check(clean, q, new, d ** -0.5, got, lse, dtype)


# ---------------------------------------------------------------------------------------------------- values that one token sees

SEEN = [
    # lens, q_heads, kv_heads, d, page, dtype, window, sinks, slots with a bad value
    ([1], 4, 2, 128, 16, BF16, 0, 0, [0]),                          # its weight is 1: nothing is left for a second part
    ([160], 4, 1, 64, 16, F16, 0, 0, [0, 77, 159]),                 # joined in a cluster
    ([500, 33], 8, 2, 128, 32, BF16, 0, 0, [5, 32]),
    ([300, 20], 80, 2, 64, 16, BF16, 0, 0, [19]),                   # one CTA to a sequence
    ([5000], 8, 1, 128, 64, F16, 0, 0, [0, 4999]),                  # parts, joined by a second kernel
    ([5000, 130], 6, 2, 64, 64, BF16, 64, 70, [3, 69, 129, 4990]),
    ([9000, 8000, 7], 16, 2, 128, 128, BF16, 0, 0, [6, 8191]),
]


@pytest.mark.parametrize("with_weights", [False, True])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan, "both"])
@pytest.mark.parametrize("lens,hq,hk,d,page,dtype,window,sinks,slots", SEEN)
def test_decode_with_values_that_are_not_finite(lens, hq, hk, d, page, dtype, window, sinks, slots, bad, with_weights):
    """An infinity that the token sees is its output's, infinities of both signs are NaN; the other channels and heads do not feel it."""
    cache = make_cache(lens, hk, d, page, dtype, fill=math.nan)
    for b, n in enumerate(lens):
        for i, slot in enumerate(s for s in slots if s < n):
            put(cache, cache.v, b, slot, math.inf if bad == "both" else bad, head=i % hk, channel=(7 * i) % d)
            put(cache, cache.v, b, slot, -math.inf if bad == "both" else bad, head=hk - 1, channel=d - 1 - i)
        if bad == "both" and slots[0] < n and n > 1:
            put(cache, cache.v, b, n - 1, -math.inf, head=0, channel=0)
    q = queries(len(lens), hq, d, dtype)
    weights = torch.zeros((len(lens), hk, cache.slots), device="cuda") if with_weights else None
    got, lse = ops.attention_paged_decode(q, cache, d ** -0.5, window=window, sinks=sinks, weights=weights)
    for b, n in enumerate(lens):
        want, want_lse, size = expect(cache, b, q[b:b + 1], torch.tensor([n - 1], device="cuda"), window, sinks, d ** -0.5)
        near(got[b:b + 1], want, U[dtype] * want.abs() + (U[dtype] ** 2 + F) * size + 1e-7, "out")
        near(lse[b:b + 1], want_lse, F * (1 + want_lse.abs()), "lse")
    if with_weights:
        assert bool(torch.isfinite(weights).all())
    assert ops.paged_cache_status() == 0


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 64)])
def test_decode_with_an_infinite_value_of_no_weight(dtype, d):
    """Where every score is minus infinity nothing is seen, infinities of V included; a small weight times infinity is infinity."""
    cache = make_cache([40], 1, d, 16, dtype)
    cache.k.zero_()
    cache.k[..., 0] = -math.inf
    put(cache, cache.v, 0, 9, math.inf, channel=2)
    q = queries(1, 2, d, dtype)
    q[..., 0] = 1.0
    got, lse = ops.attention_paged_decode(q, cache, 0.5)
    assert bool((got == 0).all()) and bool((lse == -math.inf).all())
    cache.k[..., 0] = 0.0
    put(cache, cache.k, 0, 20, 60.0, channel=0)  # a weight of e^-60 for the others
    got, _ = ops.attention_paged_decode(q, cache, 1.0)
    assert bool((got[..., 2] == math.inf).all()) and bool(torch.isfinite(got[..., 3:]).all())


# ---------------------------------------------------------------------------------------------------- values of next to no weight

@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 128), (BF16, 64), (F16, 64)])
@pytest.mark.parametrize("gap", [20.0, 60.0, 110.0])
@pytest.mark.parametrize("n,past,window,sinks", [(400, 0, 0, 0), (700, 0, 300, 5), (3, 5000, 0, 0), (300, 900, 0, 0)])
def test_prompt_with_infinite_values_of_little_weight(dtype, d, gap, n, past, window, sinks):
    """A weight of e^-gap is above 0, however 16 bits hold it: times infinity it is infinity."""
    end = n + past
    cache = make_cache([end], 2, d, 64, dtype)
    cache.k.zero_()
    for b_slot, channel, value in ((2, 3, math.inf), (133, d - 1, -math.inf), (140, 7, math.nan), (end - 140, 0, math.inf), (end - 2, 5, math.inf)):
        if 0 <= b_slot < end:
            put(cache, cache.k, 0, b_slot, -gap, channel=0)
            put(cache, cache.v, 0, b_slot, value, head=b_slot % 2, channel=channel)
    put(cache, cache.v, 0, 30, -math.inf, head=0, channel=3)  # meets the infinity of slot 2
    put(cache, cache.k, 0, 30, -gap, channel=0)
    q = torch.zeros((n, 6, d), dtype=dtype, device="cuda")
    q[..., 0] = 1.0
    got, lse = ops.attention_paged(q, cache, cu_of([n]), n, 1.0, window=window, sinks=sinks)
    check(cache, q, [n], 1.0, got, lse, dtype, window, sinks)
    again, _ = ops.attention_paged(q, cache, cu_of([n]), n, 1.0, window=window, sinks=sinks)
    assert torch.equal(again.view(torch.int16), got.view(torch.int16)) and ops.paged_cache_status() == 0


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 64)])
def test_prompt_that_sees_nothing_of_infinite_values(dtype, d):
    """Every score minus infinity: zeros, infinities of V included."""
    cache = make_cache([300], 1, d, 16, dtype)
    cache.k.zero_()
    cache.k[..., 0] = -math.inf
    put(cache, cache.v, 0, 9, math.inf, channel=2)
    put(cache, cache.v, 0, 290, math.nan, channel=3)
    q = torch.zeros((300, 2, d), dtype=dtype, device="cuda")
    q[..., 0] = 1.0
    got, lse = ops.attention_paged(q, cache, cu_of([300]), 300, 0.5)
    assert bool((lse == -math.inf).all())
    assert bool((got == 0).all())


@pytest.mark.parametrize("form", ["prompt", "decode"])
@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("n,low", [(500, 300), (20000, 12000)])
@pytest.mark.parametrize("gap", [80.0, 100.0])
def test_infinite_values_in_parts_of_little_weight(form, dtype, d, n, low, gap):
    """The slots [0, low), whole parts of the keys, have e^-gap of the others' weight: less than fp32 keeps of 1."""
    cache = make_cache([n], 1, d, 64, dtype)
    cache.k.zero_()
    for slot in range(0, low, 64):
        cache.k[cache.block_table[0, slot // 64].item(), :, :min(64, low - slot), 0] = -gap
    put(cache, cache.v, 0, 5, math.inf, channel=1)
    put(cache, cache.v, 0, low // 2, -math.inf, channel=2)
    put(cache, cache.v, 0, 8, math.inf, channel=3)
    put(cache, cache.v, 0, low // 2 + 1, -math.inf, channel=3)
    q = torch.zeros((1, 4, d), dtype=dtype, device="cuda")
    q[..., 0] = 1.0
    got, lse = ops.attention_paged(q, cache, cu_of([1]), 1, 1.0) if form == "prompt" else ops.attention_paged_decode(q, cache, 1.0)
    check(cache, q, [1], 1.0, got, lse, dtype)


# ---------------------------------------------------------------------------------------------------- eviction

@pytest.mark.parametrize("n,heads", [(60, 1), (3000, 3), (20000, 1)])
def test_evict_ranks_nan_below_minus_infinity(n, heads):
    """Of weights that are NaN in every other slot and minus infinity in the others, the latter stay; then the lowest of the NaN."""
    cache = make_cache([n], heads, 64, 16, BF16, spare=-(-(n // 2 + 7) // 16))
    weights = torch.full((1, heads, cache.slots), math.nan, device="cuda")
    weights[..., 1:n:2] = -math.inf
    used = set(cache.block_table[cache.block_table >= 0].tolist())
    table_out = torch.tensor([[p for p in range(cache.k.shape[0]) if p not in used]], dtype=torch.int32).cuda()
    for budget in (n // 2 - 5, n // 2, n // 2 + 7):
        kept, _ = ops.kv_evict(cache, weights, table_out, budget)
        want = sorted(list(range(1, n, 2))[:budget] + list(range(0, n, 2))[:max(0, budget - n // 2)])
        assert kept.tolist() == [[want] * heads]
    assert ops.paged_cache_status() == 0
