"""token_logprobs of logits far from zero, and behind scales far from one: finite numbers give finite numbers."""
import math

import pytest
import torch

from tests.test_gpu_logprobs import check, rows_of, some_targets

pytestmark = pytest.mark.gpu
bf16, f16, f32 = torch.bfloat16, torch.float16, torch.float32
INF = math.inf


def far(vocab, most, dtype):
    """Rows whose largest logit is about `most`: alike, a few alike at the top, falling by the type's steps, one on its own, ordinary ones beside a mask of it."""
    t = torch.arange(vocab, device="cuda", dtype=torch.float64)
    size = abs(most)
    step = size * torch.finfo(dtype).eps * 2
    rows = [torch.full_like(t, most), torch.where(t % 97 == 5, most, max(most - 0.5 * size, -3.38e38)), most - step * (t % 61), most - step * (vocab - 1 - t).clamp(max=60),
            torch.where(t == vocab // 2, most, max(most - size, -3.38e38)), torch.where(t % 500 == 3, t % 7, -size), torch.where(t < vocab // 2, -size, t % 5),
            torch.where(t % 3 == 0, -INF, most - step * (t % 4))]
    return torch.stack(rows).to(dtype).contiguous()


@pytest.mark.parametrize("most", [1e6, -1e6, 1.2e7, 2e7, -3e7, 1e8, 1e9, -1e9, 1.45e9, -1.45e9, 1.6e9, 1e10, -1e10, 1e20, -1e20, 1e30, -1e30, 3e38, -3e38])
@pytest.mark.parametrize("dtype", [bf16, f32], ids=["bf16", "f32"])
@pytest.mark.parametrize("vocab", [40, 8195, 70001])
def test_far_from_zero(vocab, dtype, most):
    logits = far(vocab, most, dtype)
    check(logits, some_targets(len(logits), vocab, 5), 8)
    check(logits.repeat(100, 1), some_targets(100 * len(logits), vocab, 6), 3)  # (a CTA to each row)


# (Powers of two: a scale that 32 bits hold as it is, so that a difference of large numbers is the definition's.)
@pytest.mark.parametrize("scale", [2.0 ** e for e in (20, 24, 26, 30, 40, 60, 99)], ids=str)
@pytest.mark.parametrize("dtype", [bf16, f16, f32], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("vocab", [40, 8195, 70001])
def test_scales_far_from_one(vocab, dtype, scale):
    logits = rows_of(9, vocab, dtype, seed=6).contiguous()
    logits[1] = 30.0
    logits[2] -= 200.0
    logits[3, 7:] = -INF
    logits[4] = torch.finfo(dtype).min
    logits[6, vocab // 2:] = -1e4
    check(logits, some_targets(9, vocab, 7), 8, scale)
    check(logits.repeat(80, 1), some_targets(9 * 80, vocab, 8), 2, scale)
