"""token_logprobs where fewer tokens than alternatives are numbers, or above minus infinity: the others follow by their number."""
import math

import pytest
import torch

from tests.test_gpu_logprobs import check, rows_of

pytestmark = pytest.mark.gpu
INF, NAN = math.inf, math.nan
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def allowed(rows, vocab, most, seed):
    """[rows, vocab]: 1 to `most` tokens of each row at random places."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    mask = torch.zeros(rows, vocab, dtype=torch.bool, device="cuda")
    where = torch.randint(vocab, (rows, most), generator=g, device="cuda")
    count = torch.randint(1, most + 1, (rows, 1), generator=g, device="cuda")
    return mask.scatter_(1, torch.where(torch.arange(most, device="cuda") < count, where, where[:, :1]), True)


# (1000 rows: a CTA to each, whose threads have several batches of loads. 3 rows: clusters.)
@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,vocab", [(1000, 8192), (1000, 16384), (600, 32003), (300, 70001), (3, 70001), (1, 150001)])
@pytest.mark.parametrize("none", [-INF, NAN], ids=["minus infinity", "nan"])
def test_few_are_allowed(rows, vocab, dtype, none):
    logits = rows_of(rows, vocab, dtype, seed=vocab).contiguous().masked_fill_(~allowed(rows, vocab, 6, vocab), none)
    for top in (1, 2, 5, 20, 32):
        check(logits, (torch.arange(rows, device="cuda") * 37) % vocab, top)


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("vocab", [8192, 33001])
def test_one_is_allowed_wherever_it_is(vocab, dtype):
    rows = 1000
    logits = torch.full((rows, vocab), -INF, dtype=dtype, device="cuda")
    logits[torch.arange(rows, device="cuda"), torch.arange(rows, device="cuda") * (vocab // rows) + 3] = 1.0
    check(logits, torch.arange(rows, device="cuda"), 5)
    check(logits, None, 32)


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("vocab", [4100, 16384, 32003])
def test_numbers_then_minus_infinity_then_nan(vocab, dtype):
    rows = 700
    g = torch.Generator(device="cuda").manual_seed(vocab)
    logits = torch.full((rows, vocab), NAN, dtype=dtype, device="cuda")
    logits.masked_fill_(allowed(rows, vocab, 20, 1), -INF)
    some = allowed(rows, vocab, 6, 2) & (torch.arange(rows, device="cuda") % 3 != 0)[:, None]  # (every third row has no number)
    logits = torch.where(some, torch.randn(logits.shape, generator=g, device="cuda").to(dtype), logits)
    for top in (3, 20, 32):
        check(logits, torch.arange(rows, device="cuda"), top)
