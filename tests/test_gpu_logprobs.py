"""token_logprobs against the definition in 64 bits: types, sizes, alignments, ties, masks, what is not finite."""
import math

import pytest
import torch

from owoinfer_b200 import ops

pytestmark = pytest.mark.gpu
INF, NAN = math.inf, math.nan
bf16, f16, f32 = torch.bfloat16, torch.float16, torch.float32
VIEWS = {bf16: torch.int16, f16: torch.int16, f32: torch.int32}


def exact(logits, targets, top, scale):
    """Order by the logits (NaN last, equal ones by number), values in 64 bits."""
    l = logits.double()
    # (Against the largest: next to logits of 1e38 the log of a sum has no place in 64 bits either.)
    z = l * scale
    nothing = (l == -INF).all(-1)
    most = torch.where(nothing, 0.0, z.amax(-1))
    z = z - most[:, None]
    log_sum = torch.exp(z).sum(-1).log()
    lse, z = most + log_sum, z - log_sum[:, None]
    p = torch.exp(z)
    entropy = torch.where(p > 0, -p * z, torch.where(p == 0, 0.0, p)).sum(-1)
    order = torch.sort(torch.where(l.isnan(), -INF, l), dim=-1, descending=True, stable=True)[1]
    # (NaN behind -infinity: a second stable sort by being NaN)
    last = torch.sort(l.gather(1, order).isnan().int(), dim=-1, stable=True)[1]
    order = order.gather(1, last)
    place = torch.empty_like(order).scatter_(1, order, torch.arange(l.shape[1], device=l.device).expand_as(order).contiguous())
    logprobs = ranks = None
    if targets is not None:
        t = targets.clamp(0, l.shape[1] - 1)[:, None]
        logprobs = z.gather(1, t)[:, 0]
        ranks = place.gather(1, t)[:, 0] + 1
        there = (targets >= 0) & (targets < l.shape[1])
        logprobs = torch.where(there, logprobs, torch.where(targets < 0, 0.0, NAN))
        ranks = torch.where(there, ranks, 0)
    entropy = torch.where(nothing, 0.0, entropy)
    top_tokens = order[:, :top]
    top_logprobs = z.gather(1, top_tokens)
    if targets is not None:
        logprobs = torch.where(nothing & there, -INF, logprobs)
    return logprobs, ranks, entropy, lse, torch.where(nothing[:, None], -INF, top_logprobs), top_tokens


def near(got, want, bound):
    want = want.double()
    want = torch.where(want.abs() > torch.finfo(f32).max, want.sign() * INF, want)  # (-3e38 against a largest of 3e38: fp32 has no -6e38)
    fine = want.isfinite()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.double()[~fine & ~want.isnan()], want[~fine & ~want.isnan()])
    assert ((got.double() - want).abs()[fine] <= bound.expand_as(want)[fine]).all(), (got.double() - want).abs()[fine].max()


def check(logits, targets, top, scale=1.0):
    got = ops.token_logprobs(logits, targets, top=top, scale=scale)
    logprobs, ranks, entropy, lse, top_logprobs, top_tokens = exact(logits, targets, top, scale)
    # Roundings of 2^-24: an exponent x (in binades) has two relative ones and the hardware's exponential 2^-22 of its result; weighted by 2^x that is
    # |x| 2^x <= 8 for what is up to 8 ahead of the reference, and less than 1 below it: 16 + 4. The sums are chains of vocab / 8 / 512 loads and 30
    # joins for a thread at most. What is then multiplied out has a rounding of its own size (the entropy: of the mean exponent, below 8 + log vocab).
    vocab = logits.shape[1]
    steps = 2 * (20 + 4 * vocab / 4096 / 8 + 30)
    unit = 2.0 ** -24
    bound = torch.full((len(logits),), steps * unit, dtype=torch.float64, device="cuda")
    near(got.lse, lse, bound + 4 * unit * lse.abs())
    near(got.entropy, entropy, (2 + 8 + math.log(vocab)) * bound)
    if targets is None:
        assert got.logprobs is None and got.ranks is None
    else:
        near(got.logprobs, logprobs, bound + 4 * unit * logprobs.abs())
        assert torch.equal(got.ranks.long(), ranks)
    if top == 0:
        assert got.top_tokens is None and got.top_logprobs is None
    else:
        assert torch.equal(got.top_tokens.long(), top_tokens)
        near(got.top_logprobs, top_logprobs, bound[:, None] + 4 * unit * top_logprobs.abs())


def rows_of(rows, vocab, dtype, seed=0, offset=0, std=3.0, pad=0):
    """[rows, vocab] that starts `offset` elements into its buffer, rows `vocab + pad` apart."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    flat = (std * torch.randn(offset + rows * (vocab + pad), generator=g, device="cuda")).to(dtype)
    return flat[offset:].view(rows, vocab + pad)[:, :vocab]


def some_targets(rows, vocab, seed=0):
    t = torch.randint(vocab, (rows,), generator=torch.Generator().manual_seed(seed))
    t[0] = vocab - 1
    return t.cuda()


@pytest.mark.parametrize("dtype", [bf16, f16, f32], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,vocab,top,offset,pad,scale", [
    (1, 1, 1, 0, 0, 1.0), (3, 2, 2, 1, 0, 1.0), (2, 7, 5, 3, 2, 0.5), (4, 31, 31, 0, 0, 1.0), (5, 33, 32, 5, 1, 2.0), (1, 257, 20, 7, 0, 1.0), (300, 512, 5, 0, 0, 1.0),
    (3, 4097, 32, 1, 3, 1.0), (70, 5003, 8, 2, 0, 0.7), (1, 32003, 32, 0, 0, 1.0), (2, 150001, 5, 1, 0, 1.3), (40, 65536, 20, 0, 64, 1.0), (400, 8191, 1, 3, 0, 1.0),
    (1000, 1001, 0, 0, 7, 1.0), (150, 20000, 32, 1, 1, 1e-3), (150, 20000, 3, 0, 0, 40.0),
])
def test_against_the_definition(rows, vocab, top, offset, pad, scale, dtype):
    logits = rows_of(rows, vocab, dtype, seed=vocab, offset=offset, pad=pad)
    check(logits, some_targets(rows, vocab), top, scale)


@pytest.mark.parametrize("vocab", [100, 8192, 70001])
@pytest.mark.parametrize("dtype", [bf16, f16, f32], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("top", [1, 32])
def test_ties_and_orders(vocab, dtype, top):
    t = torch.arange(vocab, device="cuda")
    kinds = [torch.zeros(vocab, device="cuda"), torch.where(t % 2 == 0, 0.0, -0.0), -t / vocab * 40.0, t / vocab * 40.0, (t % 7).float(), (t % 4096 < 40).float() * 5,
             torch.where(t % 4096 < 8, 3.0 + t / vocab, 0.0), torch.where(t >= vocab - 50, 2.0, 1.0), torch.where(t < 20, 1.0, 1.0 + (t % 3))]
    logits = torch.stack(kinds).to(dtype)
    check(logits, some_targets(len(kinds), vocab, 3), top)
    check(logits, None, top)


@pytest.mark.parametrize("vocab", [37, 5000, 64007])
@pytest.mark.parametrize("dtype", [bf16, f16, f32], ids=["bf16", "f16", "f32"])
def test_masks(vocab, dtype):
    low = torch.finfo(dtype).min
    logits = rows_of(10, vocab, dtype, seed=1, pad=3).contiguous()
    t = torch.arange(vocab, device="cuda")
    logits[0] = -INF
    logits[1, t != vocab // 2] = -INF          # one token is left
    logits[2, t % 11 != 3] = -INF
    logits[3] = low                            # as some mask: all alike
    logits[4, t != 5] = low
    logits[5, :] = low
    logits[5, vocab // 3:] = -INF              # the lowest value is still a value
    logits[6, :vocab - 2] = -INF               # the two last, outside whole loads
    logits[7, 2:] = -INF
    logits[8, : vocab // 2] = -INF             # first what weighs nothing, then the rest
    targets = torch.tensor([3, vocab // 2, 3, 7, 5, 1, vocab - 1, 30, 0, 2], device="cuda")
    for top in (0, 1, 20):
        check(logits, targets, top)
    check(logits, targets, 32, 0.25)


@pytest.mark.parametrize("vocab", [37, 9000, 64007])
@pytest.mark.parametrize("dtype", [bf16, f16, f32], ids=["bf16", "f16", "f32"])
def test_what_is_not_finite(vocab, dtype):
    logits = rows_of(7, vocab, dtype, seed=2).contiguous()
    logits[0, 11] = NAN
    logits[1, vocab - 1] = INF
    logits[2, :] = NAN
    logits[3, : vocab // 2] = NAN
    logits[4, 3:] = NAN
    logits[4, :2] = -INF
    logits[5, 30], logits[5, 31] = INF, -INF
    targets = torch.tensor([11, 5, 9, vocab - 3, 1, 31, 0], device="cuda")
    check(logits, targets, 20)


def test_targets_outside_the_vocabulary():
    logits = rows_of(5, 1000, bf16)
    check(logits, torch.tensor([-1, -100, 1000, 1 << 40, 999], device="cuda"), 3)


def test_extreme_values_and_more_candidates_than_fit():
    t = torch.arange(40000, device="cuda")
    big = torch.where(t % 3 == 0, 3e38, -3e38)
    # Loads 4096 elements of 16 bits apart belong to one thread: few threads hold every large value.
    spread = torch.where(t % 4096 < 32, 10.0 + (t // 4096) * 0.25 + (t % 32) * 1e-3, 0.0)
    few = torch.where(t % 4096 < 256, 10.0 + (t % 97) * 0.125, 0.0)
    wide = torch.where(t % 2048 < 124, 10.0 + (t % 89) * 0.125, 0.0)
    for dtype in (bf16, f32):
        check(torch.stack([big, spread, few, wide]).to(dtype).repeat(100, 1), some_targets(400, 40000), 32)
    # 31 threads have all that is above 0 between them: the bound that 32 threads reach is 0.
    check(torch.where(t % 4096 < 248, 10.0 + (t % 97) * 0.125, 0.0).to(bf16).repeat(300, 1), some_targets(300, 40000), 32)


def test_no_rows_many_rows_and_a_captured_call():
    got = ops.token_logprobs(torch.empty(0, 10, dtype=bf16, device="cuda"), top=2)
    assert got.entropy.shape == (0,) and got.top_tokens.shape == (0, 2)
    logits = rows_of(70000, 64, f16, seed=8)  # (more than a grid's second axis)
    check(logits, some_targets(70000, 64), 4)
    logits, targets = rows_of(2, 50000, bf16, seed=4), some_targets(2, 50000)
    want = ops.token_logprobs(logits, targets, top=7)
    graph, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=s):
        got = ops.token_logprobs(logits, targets, top=7)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
