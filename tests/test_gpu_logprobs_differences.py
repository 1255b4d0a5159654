"""token_logprobs where the difference of two logits passes 32 bits and, times the scale, does not."""
import math

import pytest
import torch

from tests.test_gpu_logprobs import check, rows_of, some_targets

pytestmark = pytest.mark.gpu
bf16, f16, f32 = torch.bfloat16, torch.float16, torch.float32
INF = math.inf


@pytest.mark.parametrize("scale", [1e30, 3e29, 0.25, 0.01])
def test_differences_past_the_largest_number(scale):
    logits = torch.tensor([[3e38, -3e38, -INF, 0.0, 1.0, -1.0, 2e38, -2e38] * 6], device="cuda")
    for dtype in (bf16, f32):
        check(logits.to(dtype), torch.tensor([1], device="cuda"), 30, scale)
        check(logits.to(dtype).repeat(300, 40), torch.arange(300, device="cuda"), 30, scale)


# (Powers of two: a scale that 32 bits hold as it is.)
@pytest.mark.parametrize("scale", [2.0 ** e for e in (-1, -20, -60, -99, -120, -126)], ids=str)
@pytest.mark.parametrize("dtype", [bf16, f16, f32], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("vocab", [40, 8195, 70001])
def test_small_scales(vocab, dtype, scale):
    logits = rows_of(9, vocab, dtype, seed=6).contiguous()
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    logits[3, 7:] = -INF
    logits[4] = low
    logits[5, ::2], logits[5, 1::2] = high, low
    logits[6, : vocab // 2], logits[6, vocab // 2:] = low, high
    logits[7, 2:], logits[7, :2] = -INF, high
    logits[8, ::3] = low
    check(logits, some_targets(9, vocab, 7), 8, scale)
    check(logits.repeat(80, 1), some_targets(9 * 80, vocab, 8), 2, scale)
