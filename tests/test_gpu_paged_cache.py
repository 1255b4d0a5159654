"""The operators on paged key-value caches against their definitions in 64 bits.

Tolerances. u is half a unit in the last place of the type (bf16 2^-8, fp16 2^-11, of a value's magnitude). An output is rounded once:
u * |want|. In a prompt's attention P is rounded to the type before P.V: at most u * A with A = sum p |v|; in the single-token
form bf16 P goes in as two parts: u^2 * A. What fp32 does on the way (scores of magnitude up to about 40 with relative errors of some
2^-22, the exponential's 2^-22, sums) stays below F * A with F = 2e-5, and below F in the logarithm of the sum.
"""
import math

import pytest
import torch

from owoinfer_b200 import ops

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
U = {BF16: 2.0 ** -8, F16: 2.0 ** -11}
F = 2e-5


@pytest.fixture(autouse=True)
def _clean_status():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    ops.paged_cache_status(clear=True)
    yield
    torch.cuda.synchronize()


def make_cache(lens, kv_heads, d, page, dtype, seed=1, rows_outside=False, spare=2, fill=None, width=None):
    """A cache with pages in random order. rows_outside: pools laid out [pages, page, heads, d]. fill: what unused slots hold."""
    g = torch.Generator().manual_seed(seed)
    need = [(n + page - 1) // page for n in lens]
    pages = sum(need) + spare
    shape = (pages, page, kv_heads, d) if rows_outside else (pages, kv_heads, page, d)
    pools = [torch.randn(shape, generator=g).to(dtype).cuda() for _ in range(2)]
    if rows_outside:
        pools = [p.permute(0, 2, 1, 3) for p in pools]
    order = torch.randperm(pages, generator=g).to(torch.int32)
    width = max(max(need), 1) if width is None else width
    table, at = torch.full((len(lens), width), -1, dtype=torch.int32), 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    if fill is not None:
        used = torch.zeros((pages, page), dtype=torch.bool)
        for i, n in enumerate(lens):
            for j in range(n):
                used[table[i, j // page], j % page] = True
        for p in pools:
            p.masked_fill_(~used[:, None, :, None].cuda(), fill)
    return ops.PagedCache(pools[0], pools[1], table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda())


def rows_of(cache, pool, b, n):
    at = torch.arange(n, device="cuda")
    return pool[cache.block_table[b].long()[at // cache.page_size], :, at % cache.page_size]  # [n, heads, d]


def cu_of(counts):
    return torch.tensor([0] + list(counts), dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()


def seen_of(slots, n, window, sinks):
    key = torch.arange(n, device="cuda")
    seen = key[None] <= slots[:, None]
    return seen & ((key[None] < sinks) | (slots[:, None] - key[None] < window)) if window else seen


def attention_64(q, k, v, seen, scale):
    """q [n, heads, d], k, v [slots, kv_heads, d]; (out, lse, sum p |v|, p) with p [heads, n, slots]. What is not seen plays no part."""
    group = q.shape[1] // k.shape[1]
    s = torch.einsum("nhd,jhd->hnj", q.double(), k.double().repeat_interleave(group, 1)) * scale
    s = torch.where(seen[None], s, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.where(seen[None], (s - lse[..., None]).exp(), 0.0)
    vv = v.double().repeat_interleave(group, 1)
    # (0 * infinity: a slot that is not seen is left out of the product)
    fine = torch.where(torch.isfinite(vv), vv, 0.0)
    out, size = torch.einsum("hnj,jhd->nhd", p, fine), torch.einsum("hnj,jhd->nhd", p, fine.abs())
    odd = (~torch.isfinite(vv)).any(-1).any(-1).nonzero()[:, 0].tolist()
    for j in odd:
        out += torch.where(seen[:, j][:, None, None] & ~torch.isfinite(vv[j])[None], vv[j][None], 0.0)
    return out, lse.transpose(0, 1), size, p


def near(got, want, bound, what):
    got, want = got.double(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), what
    over = ((got - want).abs() - bound)[fine]
    assert over.numel() == 0 or over.max().item() <= 0, (what, over.max().item())


# ---------------------------------------------------------------------------------------------------- append

def append_64(x, weight, sin, cos, interleaved, eps):
    """x [n, heads, d] in 64 bits; also the sizes that the rounding goes by."""
    if weight is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    size = x.abs()
    if sin is not None:
        half = sin.shape[-1]
        a = torch.arange(0, 2 * half, 2) if interleaved else torch.arange(half)
        b = a + (1 if interleaved else half)
        y, size = x.clone(), size.clone()
        y[..., a] = x[..., a] * cos[:, None] - x[..., b] * sin[:, None]
        y[..., b] = x[..., b] * cos[:, None] + x[..., a] * sin[:, None]
        size[..., a] = size[..., b] = x[..., a].abs() + x[..., b].abs()
        x = y
    return x, size


APPEND = [
    # lens, new, q_heads, kv_heads, d, page, dtype, rot, interleaved, norm, positions, rows_outside
    ([1], [1], 1, 1, 64, 16, BF16, 64, False, True, None, False),
    ([17], [17], 4, 2, 128, 16, BF16, 128, False, True, None, False),
    ([40, 1, 0, 33], [3, 1, 0, 33], 5, 1, 128, 32, F16, 64, False, True, 1000, False),
    ([100, 0, 65], [64, 0, 2], 7, 3, 64, 64, BF16, 32, True, True, 5, True),
    ([9], [9], 2, 2, 128, 128, F16, 128, True, False, None, False),
    ([300] * 37, [1] * 37, 32, 8, 128, 16, BF16, 128, False, True, 77, False),
    ([5, 6], [5, 6], 3, 1, 64, 16, F16, 0, False, True, None, True),
    ([8] * 300, [1] * 300, 2, 1, 64, 16, BF16, 16, False, False, None, False),
    ([700, 3], [690, 3], 16, 4, 128, 256, BF16, 96, False, True, None, False),
]


@pytest.mark.parametrize("lens,new,hq,hk,d,page,dtype,rot,interleaved,norm,shift,outside", APPEND)
def test_append(lens, new, hq, hk, d, page, dtype, rot, interleaved, norm, shift, outside):
    cache = make_cache(lens, hk, d, page, dtype, rows_outside=outside)
    before = cache.k.clone(), cache.v.clone()
    g = torch.Generator().manual_seed(3)
    tokens, eps = sum(new), 1e-5
    wide = torch.randn((tokens, (hq + 2 * hk) * d + 16), generator=g).to(dtype).cuda()
    qkv = wide[:, 8:-8]
    wq, wk = [(1 + 0.2 * torch.randn(d, generator=g)).to(dtype).cuda() if norm else None for _ in range(2)]
    slots = [end - n + i for end, n in zip(lens, new) for i in range(n)]
    positions = None if shift is None else torch.tensor([s + shift for s in slots], dtype=torch.int32).cuda()
    rope = torch.randn((max(lens) + (shift or 0), rot), generator=g).cuda() if rot else None
    got = ops.qk_norm_rope_append(qkv, cache, cu_of(new), wq, wk, rope, positions=positions, eps=eps, interleaved=interleaved)
    x = qkv.double().view(tokens, hq + 2 * hk, d)
    sin = cos = None
    if rot:
        at = torch.tensor(slots).cuda() + (shift or 0)
        sin, cos = rope[at].double().split(rot // 2, -1)
    want_q, size_q = append_64(x[:, :hq], wq, sin, cos, interleaved, eps)
    want_k, size_k = append_64(x[:, hq:hq + hk], wk, sin, cos, interleaved, eps)
    bound = lambda want, size: U[dtype] * want.abs() + F * size + 1e-7  # noqa: E731 (fp16 subnormals: 2^-25)
    near(got, want_q, bound(want_q, size_q), "q")
    k, v, at = before[0].double(), before[1].clone(), 0
    touched = torch.zeros(k.shape[0], page, dtype=torch.bool, device="cuda")
    size = torch.zeros_like(k)
    for b, (end, n) in enumerate(zip(lens, new)):
        for i in range(n):
            slot = end - n + i
            place = cache.block_table[b, slot // page].item(), slice(None), slot % page
            k[place], size[place], v[place] = want_k[at], size_k[at], qkv.view(tokens, -1, d)[at, hq + hk:] if qkv.is_contiguous() else x[at, hq + hk:].to(dtype)
            touched[place[0], place[2]] = True
            at += 1
    near(cache.k, k, bound(k, size) * touched[:, None, :, None], "k")  # (bound 0: not touched)
    assert torch.equal(cache.v, v)
    assert ops.paged_cache_status() == 0


def test_append_in_place_of_the_projection():
    cache = make_cache([50, 20], 2, 128, 16, BF16)
    qkv = torch.randn(7, 10 * 128, generator=torch.Generator().manual_seed(1)).to(BF16).cuda()
    w = torch.ones(128, dtype=BF16, device="cuda")
    rope = torch.randn(64, 128).cuda()
    want = ops.qk_norm_rope_append(qkv, cache, cu_of([4, 3]), w, w, rope)
    k = cache.k.clone()
    view = qkv.view(7, 10, 128)[:, :6]
    got = ops.qk_norm_rope_append(qkv, cache, cu_of([4, 3]), w, w, rope, out=view)
    assert torch.equal(got, want) and got.data_ptr() == qkv.data_ptr() and torch.equal(cache.k, k)


# ---------------------------------------------------------------------------------------------------- a prompt's attention

PROMPT = [
    # lens, new, q_heads, kv_heads, d, page, dtype, window, sinks, rows_outside
    ([1], [1], 1, 1, 64, 16, BF16, 0, 0, False),
    ([2], [2], 1, 1, 128, 16, BF16, 0, 0, False),
    ([130], [130], 2, 2, 128, 16, BF16, 0, 0, False),       # one query head to a key head: the edge runs through three tiles
    ([257], [257], 3, 3, 64, 32, F16, 0, 0, True),
    ([1000, 127, 0, 128, 129], [1000, 127, 0, 128, 129], 4, 1, 128, 64, BF16, 0, 0, False),
    ([700, 60], [5, 60], 16, 1, 128, 128, BF16, 0, 0, False),
    ([640], [333], 14, 2, 64, 256, F16, 0, 0, False),
    ([3, 300], [10, 310], 6, 2, 128, 16, BF16, 0, 0, False),  # fewer slots than tokens: the first tokens see nothing
    ([0, 40], [4, 40], 4, 4, 64, 16, BF16, 0, 0, False),
    ([900], [900], 8, 2, 128, 32, BF16, 100, 4, False),
    ([900], [900], 2, 2, 64, 32, F16, 1, 0, False),
    ([1500], [700], 4, 2, 128, 64, BF16, 256, 130, False),
    ([1500], [700], 4, 2, 128, 64, BF16, 257, 0, True),
    ([600], [600], 5, 1, 128, 16, F16, 5000, 9, False),
    ([520], [130], 33, 1, 64, 16, BF16, 64, 600, False),
]


def check_prompt(cache, q, new, window, sinks, scale, got, lse, dtype):
    at = 0
    for b, n in enumerate(new):
        end = int(cache.seq_lens[b])
        if n == 0:
            continue
        slots = torch.arange(end - n, end, device="cuda")
        if end == 0:
            assert torch.equal(got[at:at + n], torch.zeros_like(got[at:at + n])) and bool((lse[at:at + n] == -math.inf).all())
            at += n
            continue
        seen = seen_of(slots, end, window, sinks)
        want, want_lse, size, _ = attention_64(q[at:at + n], rows_of(cache, cache.k, b, end), rows_of(cache, cache.v, b, end), seen, scale)
        none = ~seen.any(1)
        want[none], size[none] = 0.0, 0.0
        near(got[at:at + n], want, U[dtype] * want.abs() + (U[dtype] + F) * size + 1e-7, "out")
        near(lse[at:at + n], want_lse, F * (1 + want_lse.abs().nan_to_num(posinf=0)), "lse")
        at += n


@pytest.mark.parametrize("lens,new,hq,hk,d,page,dtype,window,sinks,outside", PROMPT)
def test_prompt(lens, new, hq, hk, d, page, dtype, window, sinks, outside):
    # What unused slots hold must not matter.
    cache = make_cache(lens, hk, d, page, dtype, rows_outside=outside, fill=math.nan)
    g = torch.Generator().manual_seed(5)
    wide = (2.0 * torch.randn((sum(new), hq + 2, d), generator=g)).to(dtype).cuda()
    q = wide[:, 1:-1]
    out = torch.full((sum(new), hq + 1, d), 7.0, dtype=dtype, device="cuda")
    scale = d ** -0.5
    got, lse = ops.attention_paged(q, cache, cu_of(new), max(new), scale, window=window, sinks=sinks, out=out[:, 1:])
    check_prompt(cache, q, new, window, sinks, scale, got, lse, dtype)
    assert bool((out[:, 0] == 7.0).all()) and ops.paged_cache_status() == 0
    again, _ = ops.attention_paged(q, cache, cu_of(new), max(new), scale, window=window, sinks=sinks)
    assert torch.equal(again.view(torch.int16), got.contiguous().view(torch.int16))


@pytest.mark.parametrize("lens,new,hq,hk,d,page,dtype,window,sinks", [
    ([5000], [1], 8, 1, 128, 16, BF16, 0, 0),
    ([6000, 0, 700], [3, 0, 300], 10, 2, 64, 64, F16, 0, 0),
    ([6000, 5], [300, 9], 4, 1, 128, 32, BF16, 0, 0),         # a short sequence has parts without keys, and tokens that see nothing
    ([9000], [130], 7, 1, 128, 128, BF16, 2500, 700),
])
@pytest.mark.parametrize("bad", [0.5, math.nan, math.inf])
def test_prompt_over_a_long_cache(lens, new, hq, hk, d, page, dtype, window, sinks, bad):
    """Few tokens over many slots: the keys are cut into parts that are worked on apart."""
    cache = make_cache(lens, hk, d, page, dtype, fill=math.nan)
    assert ops.attention_paged_workspace_bytes(cache, sum(new), hq, max(new), window, sinks) > 256
    for slot in (lens[0] - 1, lens[0] - 2, lens[0] - 140):  # near the causal edge, where some rows do not see them
        if slot < lens[0] - new[0] + 1 or bad == 0.5:
            continue
        cache.v[cache.block_table[0, slot // page].item(), 0, slot % page, 3] = bad
    q = (2.0 * torch.randn((sum(new), hq, d), generator=torch.Generator().manual_seed(5))).to(dtype).cuda()
    got, lse = ops.attention_paged(q, cache, cu_of(new), max(new), d ** -0.5, window=window, sinks=sinks)
    check_prompt(cache, q, new, window, sinks, d ** -0.5, got, lse, dtype)
    again, _ = ops.attention_paged(q, cache, cu_of(new), max(new), d ** -0.5, window=window, sinks=sinks)
    assert torch.equal(again.view(torch.int16), got.view(torch.int16)) and ops.paged_cache_status() == 0


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("steep", [3.0, 30.0])
def test_prompt_with_scores_that_rise(dtype, steep):
    """Every key tile outdoes the one before by far: the reference has to be raised, and the output scaled, again and again."""
    n, d = 900, 128
    cache = make_cache([n], 2, d, 16, dtype)
    up = torch.linspace(0.0, steep, n).to(dtype).cuda()
    for j in range(n):
        cache.k[cache.block_table[0, j // 16].item(), :, j % 16, 0] = up[j]
    q = torch.randn((n, 4, d), generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
    q[:, :, 0] = 40.0
    scale = 0.25
    got, lse = ops.attention_paged(q, cache, cu_of([n]), n, scale)
    k, v = rows_of(cache, cache.k, 0, n), rows_of(cache, cache.v, 0, n)
    want, want_lse, size, _ = attention_64(q, k, v, seen_of(torch.arange(n, device="cuda"), n, 0, 0), scale)
    # Scores of up to 300: fp32 keeps them to about 300 * 2^-22 = 7e-5, which the weights have as a relative error.
    slack = F + 40.0 * steep * scale * 2.0 ** -21
    near(got, want, U[dtype] * want.abs() + (U[dtype] + slack) * size, "out")
    near(lse, want_lse, slack * (1 + want_lse.abs()), "lse")


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_prompt_keeps_hidden_infinities_out(dtype, d, bad):
    """Keys and values that are not finite reach the rows that see them, and no others."""
    n, window, sinks = 500, 90, 3
    cache = make_cache([n], 2, d, 32, dtype)
    q = torch.randn((n, 6, d), generator=torch.Generator().manual_seed(9)).to(dtype).cuda()
    for slot, channel in ((0, 5), (130, 0), (258, 40), (259, 40), (499, d - 1)):
        cache.v[cache.block_table[0, slot // 32].item(), slot % 2, slot % 32, channel] = bad
    if bad != math.inf:
        cache.v[cache.block_table[0, 9].item(), 0, 300 % 32, 40] = math.inf  # slot 300: infinities of both signs meet
    got, lse = ops.attention_paged(q, cache, cu_of([n]), n, d ** -0.5, window=window, sinks=sinks)
    check_prompt(cache, q, [n], window, sinks, d ** -0.5, got, lse, dtype)
    got, lse = ops.attention_paged(q, cache, cu_of([n]), n, d ** -0.5)
    # (Without a window slots 0, 130 ... lie in tiles that later rows see whole: there an infinity meets every weight, none of them 0.)
    check_prompt(cache, q, [n], 0, 0, d ** -0.5, got, lse, dtype)
    # A key that is not finite: rows that do not see it are as before.
    clean = make_cache([n], 2, d, 32, dtype)
    want, _ = ops.attention_paged(q, clean, cu_of([n]), n, d ** -0.5)
    clean.k[clean.block_table[0, 300 // 32].item(), 0, 300 % 32] = bad
    got, _ = ops.attention_paged(q, clean, cu_of([n]), n, d ** -0.5)
    assert torch.equal(got[:300], want[:300]) and torch.equal(got[:, 3:], want[:, 3:])
    assert not bool(torch.isfinite(got[300:, :3]).all(-1).any()) if math.isnan(bad) else True


# ---------------------------------------------------------------------------------------------------- one token

DECODE = [
    # lens, q_heads, kv_heads, d, page, dtype, window, sinks, rows_outside
    ([1], 1, 1, 64, 16, BF16, 0, 0, False),
    ([0, 1, 15, 16, 17, 31, 64, 65], 4, 2, 128, 16, BF16, 0, 0, False),
    ([1000, 0, 999, 3], 8, 1, 128, 32, BF16, 0, 0, True),
    ([5000], 7, 1, 64, 64, F16, 0, 0, False),
    ([5000, 4097], 16, 2, 128, 128, BF16, 0, 0, False),
    ([777], 17, 1, 128, 16, F16, 0, 0, False),               # more query heads than an MMA has rows
    ([300, 20], 80, 2, 64, 16, BF16, 0, 0, False),
    ([5000, 10, 200], 8, 4, 128, 16, BF16, 129, 0, False),
    ([5000, 130, 0], 6, 2, 64, 64, F16, 64, 70, True),
    ([3000], 5, 5, 128, 16, BF16, 1, 1, False),
    ([3000], 4, 1, 128, 1024, BF16, 2000, 3000, False),
]


def check_decode(cache, q, window, sinks, scale, got, lse, dtype, weights=None, weights_out=None, untouched=None):
    hq, hk = q.shape[1], cache.kv_heads
    for b in range(cache.batch):
        end = int(cache.seq_lens[b])
        if end == 0:
            assert bool((got[b] == 0).all()) and bool((lse[b] == -math.inf).all())
        else:
            seen = seen_of(torch.tensor([end - 1], device="cuda"), end, window, sinks)
            want, want_lse, size, p = attention_64(q[b:b + 1], rows_of(cache, cache.k, b, end), rows_of(cache, cache.v, b, end), seen, scale)
            near(got[b:b + 1], want, U[dtype] * want.abs() + (2.0 ** -16 if dtype == BF16 else U[dtype]) * size + F * size + 1e-7, "out")
            near(lse[b:b + 1], want_lse, F * (1 + want_lse.abs()), "lse")
        if weights is not None:
            want = untouched[b].double()
            if end:
                got_of = p[:, 0].view(hk, hq // hk, end).sum(1)
                before = weights[b, :, :end].double().clone()
                before[:, end - 1] = 0.0
                near(weights_out[b, :, :end], before + got_of, F * got_of + 2.0 ** -23 * (before + got_of).abs(), "weights")
            assert torch.equal(weights_out[b, :, end:].double(), want[:, end:])


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (BF16, 64), (F16, 64)])
@pytest.mark.parametrize("window", [0, 64])
def test_prompt_keeps_the_largest_hidden_values_out(dtype, d, window):
    """What is not seen has a weight of 0, not of the smallest number: times the type's largest value that would be a value like any other."""
    cache = make_cache([300], 2, d, 32, dtype)
    q = torch.randn((300, 8, d), generator=torch.Generator().manual_seed(5)).to(dtype).cuda()
    place = (cache.block_table[0, 192 // 32].item(), slice(None), slice(0, 16))  # slots 192 to 207
    outs = []
    for value in (0.0, torch.finfo(dtype).max, torch.finfo(dtype).min):
        cache.v[place] = value
        got, _ = ops.attention_paged(q, cache, cu_of([300]), 300, d ** -0.5, window=window)
        outs.append(torch.cat([got[:192], got[207 + window:] if window else got[:0]]))
    assert torch.equal(outs[1], outs[0]) and torch.equal(outs[2], outs[0])


@pytest.mark.parametrize("with_weights", [False, True])
@pytest.mark.parametrize("lens,hq,hk,d,page,dtype,window,sinks,outside", DECODE)
def test_decode(lens, hq, hk, d, page, dtype, window, sinks, outside, with_weights):
    cache = make_cache(lens, hk, d, page, dtype, rows_outside=outside, fill=math.nan)
    g = torch.Generator().manual_seed(6)
    q = (2.0 * torch.randn((len(lens), hq + 1, d), generator=g)).to(dtype).cuda()[:, 1:]
    weights = weights_out = untouched = None
    if with_weights:
        weights = torch.rand((len(lens), hk, cache.slots + 3), generator=g).cuda()
        for b, n in enumerate(lens):
            if n:
                weights[b, :, n - 1] = math.nan  # the newest slot's is not read
        weights_out = torch.full_like(weights, 5.0)
        untouched = weights_out.clone()
    scale = d ** -0.5
    out = torch.full((len(lens), hq + 1, d), 7.0, dtype=dtype, device="cuda")
    got, lse = ops.attention_paged_decode(q, cache, scale, window=window, sinks=sinks, weights=weights, weights_out=weights_out, out=out[:, :-1])
    check_decode(cache, q, window, sinks, scale, got, lse, dtype, weights, weights_out, untouched)
    assert bool((out[:, -1] == 7.0).all()) and ops.paged_cache_status() == 0
    again, _ = ops.attention_paged_decode(q, cache, scale, max_len=max(max(lens), 1), window=window, sinks=sinks)
    check_decode(cache, q, window, sinks, scale, again, lse, dtype)
    if with_weights:  # in place, and the same bits every time
        ops.attention_paged_decode(q, cache, scale, window=window, sinks=sinks, weights=weights)
        for b, n in enumerate(lens):
            assert torch.equal(weights[b, :, :n], weights_out[b, :, :n])


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_decode_keeps_hidden_infinities_out(bad):
    n, window, sinks = 700, 50, 2
    cache = make_cache([n], 2, 128, 16, BF16)
    q = torch.randn((1, 8, 128), generator=torch.Generator().manual_seed(4)).to(BF16).cuda()
    want, want_lse = ops.attention_paged_decode(q, cache, 0.1, window=window, sinks=sinks)
    for slot in (2, 3, 15, 16, 400, 640, 649):  # next to what is seen, in the same pages
        for pool in (cache.k, cache.v):
            pool[cache.block_table[0, slot // 16].item(), :, slot % 16] = bad
    weights = torch.zeros((1, 2, cache.slots), device="cuda")
    got, lse = ops.attention_paged_decode(q, cache, 0.1, window=window, sinks=sinks, weights=weights)
    near(got, want.double(), 2 * U[BF16] * want.double().abs() + 1e-7, "out")
    near(lse, want_lse.double(), F * (1 + want_lse.double().abs()), "lse")
    assert bool(torch.isfinite(weights).all()) and abs(float(weights.sum()) - 8.0) < 1e-4


def test_decode_with_scores_that_rise():
    n, d = 4000, 64
    for dtype in (BF16, F16):
        cache = make_cache([n], 1, d, 16, dtype)
        for j in range(0, n, 16):
            cache.k[cache.block_table[0, j // 16].item(), 0, :, 0] = 30.0 * j / n
        q = torch.randn((1, 3, d), generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
        q[:, :, 0] = 30.0
        got, lse = ops.attention_paged_decode(q, cache, 0.25)
        want, want_lse, size, _ = attention_64(q, rows_of(cache, cache.k, 0, n), rows_of(cache, cache.v, 0, n), seen_of(torch.tensor([n - 1], device="cuda"), n, 0, 0), 0.25)
        slack = F + 225.0 * 2.0 ** -21
        near(got, want, U[dtype] * want.abs() + (2.0 ** -16 if dtype == BF16 else U[dtype]) * size + slack * size, "out")
        near(lse, want_lse, slack * (1 + want_lse.abs()), "lse")


def test_one_token_through_both_forms():
    lens = [1, 100, 2000]
    cache = make_cache(lens, 2, 128, 32, BF16)
    q = torch.randn((3, 8, 128), generator=torch.Generator().manual_seed(8)).to(BF16).cuda()
    a, lse_a = ops.attention_paged(q, cache, cu_of([1, 1, 1]), 1, 0.09, window=700, sinks=4)
    b, lse_b = ops.attention_paged_decode(q, cache, 0.09, window=700, sinks=4)
    assert (a.double() - b.double()).norm() <= 3 * U[BF16] * b.double().norm() and (lse_a - lse_b).abs().max() <= 2 * F * (1 + lse_b.abs().max())


# ---------------------------------------------------------------------------------------------------- eviction

def kept_of(weights, n, sinks, recent, budget):
    if n <= budget:
        return list(range(n))
    rank = [(-w if w == w else math.inf, j) for j, w in enumerate(weights)][sinks:n - recent]
    return list(range(sinks)) + sorted(j for _, j in sorted(rank)[:budget - sinks - recent]) + list(range(n - recent, n))


EVICT = [
    # lens, kv_heads, d, page, dtype, sinks, recent, budget, weights, rows_outside
    ([40], 1, 64, 16, BF16, 0, 0, 1, "random", False),
    ([100, 10, 0, 33, 32], 2, 128, 16, BF16, 2, 8, 32, "random", False),
    ([100, 64], 3, 64, 32, F16, 10, 22, 32, "random", True),       # nothing between is kept
    ([500, 301], 2, 128, 64, BF16, 4, 50, 300, "equal", False),
    ([500], 2, 128, 16, BF16, 0, 0, 77, "few", False),
    ([500], 1, 64, 16, BF16, 3, 0, 100, "odd", False),
    ([700, 3, 0], 8, 128, 32, BF16, 4, 30, 200, "random", True),    # many heads, few slots
    ([3000], 2, 128, 64, BF16, 4, 500, 2100, "few", False),        # few heads, many slots that stay
    ([9000, 8193], 2, 64, 128, F16, 4, 100, 4000, "few", False),   # two CTAs to a head
    ([70000], 1, 64, 256, BF16, 4, 1000, 20001, "random", False),  # the most CTAs, more than one round of each
    ([70000, 69999], 1, 64, 256, BF16, 0, 0, 65537, "few", False),
]


@pytest.mark.parametrize("lens,hk,d,page,dtype,sinks,recent,budget,kind,outside", EVICT)
def test_evict(lens, hk, d, page, dtype, sinks, recent, budget, kind, outside):
    batch, pages_out = len(lens), (budget + page - 1) // page
    cache = make_cache(lens, hk, d, page, dtype, rows_outside=outside, spare=batch * pages_out + 1)
    g = torch.Generator().manual_seed(11)
    used = set(cache.block_table[cache.block_table >= 0].tolist())
    free = [p for p in range(cache.k.shape[0]) if p not in used]
    table_out = torch.tensor(free[:batch * pages_out], dtype=torch.int32).view(batch, pages_out).cuda()
    shape = (batch, hk, cache.slots)
    weights = torch.randn(shape, generator=g).exp()
    if kind == "equal":
        weights = torch.ones(shape)
    if kind == "few":
        weights = torch.randint(0, 3, shape, generator=g).float()
    if kind == "odd":  # NaN below everything, zeros of both signs alike, infinities, negative values
        values = torch.tensor([math.nan, 0.0, -0.0, math.inf, -math.inf, -1.0, 1e-42, 3.0])
        weights = values[torch.randint(0, len(values), shape, generator=g)]
    k, v = cache.k.clone(), cache.v.clone()
    weights_out = torch.full((batch, hk, budget + 5), 9.0, device="cuda")
    kept, lens_out = ops.kv_evict(cache, weights.cuda(), table_out, budget, sinks=sinks, recent=recent, weights_out=weights_out)
    assert lens_out.tolist() == [min(n, budget) for n in lens]
    want_w = torch.full_like(weights_out, 9.0)
    for b, n in enumerate(lens):
        for h in range(hk):
            want = kept_of(weights[b, h].tolist(), n, sinks, recent, budget)
            assert kept[b, h].tolist() == want + [-1] * (budget - len(want)), (b, h)
            at, to = torch.tensor(want, dtype=torch.long).cuda(), torch.arange(len(want), device="cuda")
            want_w[b, h, :len(want)] = weights[b, h].cuda()[at]
            source, place = cache.block_table[b].long()[at // page], table_out[b].long()[to // page]
            k[place, h, to % page], v[place, h, to % page] = k[source, h, at % page], v[source, h, at % page]
    assert torch.equal(cache.k, k) and torch.equal(cache.v, v)
    assert torch.equal(weights_out.view(torch.int32), want_w.view(torch.int32))
    assert ops.paged_cache_status() == 0
    again, _ = ops.kv_evict(cache, weights.cuda(), table_out, budget, sinks=sinks, recent=recent)
    assert torch.equal(again, kept)


# ---------------------------------------------------------------------------------------------------- bounds, streams, graphs, size

def test_what_lies_outside_is_left_out_and_reported():
    cache = make_cache([100, 100], 2, 128, 16, BF16, spare=8)
    q = torch.randn((2, 4, 128), device="cuda").to(BF16)
    good, _ = ops.attention_paged_decode(q, cache, 0.1)
    table = cache.block_table
    table[1, 3] = 10 ** 6
    got, _ = ops.attention_paged_decode(q, cache, 0.1)
    prompt, _ = ops.attention_paged(q, cache, cu_of([1, 1]), 1, 0.1)
    assert torch.equal(got[0], good[0]) and bool(torch.isfinite(got).all()) and bool(torch.isfinite(prompt).all())
    assert (prompt[1].double() - got[1].double()).norm() <= 3 * U[BF16] * got[1].double().norm()  # both read zeros there
    assert ops.paged_cache_status(clear=True) == 1
    table[1, 3] = -5
    ops.kv_evict(cache, torch.rand((2, 2, cache.slots), device="cuda"), table[:, :4].flip(0).contiguous(), 64)
    assert ops.paged_cache_status(clear=True) == 1
    cache.seq_lens[0], cache.seq_lens[1], table[1, 3] = 10 ** 9, -3, 0
    got, lse = ops.attention_paged_decode(q, cache, 0.1)
    assert bool(torch.isfinite(got).all()) and bool((got[1] == 0).all()) and bool((lse[1] == -math.inf).all())
    assert ops.paged_cache_status(clear=True) == 2
    cache.seq_lens.fill_(100)
    ops.attention_paged_decode(q, cache, 0.1, max_len=50)
    assert ops.paged_cache_status(clear=True) == 2
    for cu in ([0, 3, 1], [0, -1, 2], [0, 1, 900]):
        ops.attention_paged(q, cache, torch.tensor(cu, dtype=torch.int32).cuda(), 2, 0.1)
        assert ops.paged_cache_status(clear=True) & 4
    qkv = torch.randn((3, 8 * 128), device="cuda").to(BF16)
    rope = torch.randn((50, 128), device="cuda")
    cache.seq_lens[0] = 1
    k = cache.k.clone()
    ops.qk_norm_rope_append(qkv, cache, cu_of([3, 0]), None, None, rope)  # three tokens for one slot
    assert ops.paged_cache_status(clear=True) == 4
    changed = (cache.k != k).any(-1).any(1).nonzero().tolist()
    assert changed == [[int(table[0, 0]), 0]]
    ops.qk_norm_rope_append(qkv, cache, cu_of([0, 3]), None, None, rope)  # slots 97 to 99 of a table of 50 positions
    assert ops.paged_cache_status(clear=True) == 8
    assert ops.paged_cache_status() == 0


def test_on_another_stream_and_replayed_from_a_graph():
    cache = make_cache([200, 77], 2, 128, 16, BF16, width=40, spare=80)
    spare = [p for p in range(cache.k.shape[0]) if p not in set(cache.block_table[cache.block_table >= 0].tolist())]
    q = torch.randn((2, 8, 128), device="cuda").to(BF16)
    qkv = torch.randn((2, 12 * 128), device="cuda").to(BF16)
    w, rope, cu = torch.ones(128, dtype=BF16, device="cuda"), torch.randn((700, 128), device="cuda"), cu_of([1, 1])
    weights = torch.zeros((2, 2, cache.slots), device="cuda")
    weights_out = torch.zeros_like(weights)

    def step():
        new_q = ops.qk_norm_rope_append(qkv, cache, cu, w, w, rope)
        out, lse = ops.attention_paged_decode(new_q, cache, 0.1, weights=weights, weights_out=weights_out)
        prompt, _ = ops.attention_paged(new_q, cache, cu, 1, 0.1, window=64, sinks=1)
        return out, lse, prompt

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = step()
    torch.cuda.current_stream().wait_stream(side)
    for grown in (0, 1, 130):  # the lengths are read when the graph runs
        lens = torch.tensor([200 + grown, 77 + grown], dtype=torch.int32).cuda()
        for b, n in enumerate(lens.tolist()):
            for i in range((n + 15) // 16):
                if int(cache.block_table[b, i]) < 0:
                    cache.block_table[b, i] = spare.pop()
        cache.seq_lens.copy_(lens)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert ops.paged_cache_status() == 0


def test_offsets_past_32_bits():
    """A pool of 2^31 elements and more: the pages in use lie at its end."""
    hk, d, page = 8, 128, 64
    pages = 2 ** 31 // (hk * d * page) + 40
    if torch.cuda.mem_get_info()[0] < 6 * pages * hk * d * page:
        pytest.skip("needs about 13 GB")
    k, v = (torch.zeros((pages, hk, page, d), dtype=BF16, device="cuda") for _ in range(2))
    n = 1000
    table = torch.arange(pages - 16, pages, dtype=torch.int32).cuda()[None].contiguous()
    cache = ops.PagedCache(k, v, table, torch.tensor([n], dtype=torch.int32).cuda())
    small = ops.PagedCache(torch.zeros((16, hk, page, d), dtype=BF16, device="cuda"), torch.zeros((16, hk, page, d), dtype=BF16, device="cuda"),
                           torch.arange(16, dtype=torch.int32).cuda()[None].contiguous(), cache.seq_lens)
    qkv = torch.randn((n, 32 * d), generator=torch.Generator().manual_seed(1)).to(BF16).cuda()
    w, rope = torch.ones(d, dtype=BF16, device="cuda"), torch.randn((n, d), generator=torch.Generator().manual_seed(2)).cuda()
    outs = []
    for c in (cache, small):
        q = ops.qk_norm_rope_append(qkv, c, cu_of([n]), w, w, rope)
        weights = torch.zeros((1, hk, c.slots), device="cuda")
        a, _ = ops.attention_paged(q, c, cu_of([n]), n, 0.1)
        b, _ = ops.attention_paged_decode(q[-1:], c, 0.1, weights=weights)
        outs.append((q, a, b, weights))
    assert all(torch.equal(x, y) for x, y in zip(*outs)) and torch.equal(k[-16:], small.k) and torch.equal(v[-16:], small.v)
    out = torch.arange(pages - 20, pages - 16, dtype=torch.int32).cuda()[None].contiguous()
    kept, _ = ops.kv_evict(cache, outs[0][3], out, 200, sinks=4, recent=50)
    at = kept[0, 3].long()
    assert torch.equal(k[-20:-16, 3].reshape(-1, d)[:200], small.k[:, 3].reshape(-1, d)[at])
    assert ops.paged_cache_status() == 0
