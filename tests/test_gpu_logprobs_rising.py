"""token_logprobs where a row's larger logits come after many smaller ones, away from zero: what was summed up first keeps its weight."""
import pytest
import torch

from tests.test_gpu_logprobs import check, some_targets

pytestmark = pytest.mark.gpu


# (500 rows: a CTA to each, whose threads see several batches of loads one after the other. 2 rows: clusters.)
@pytest.mark.parametrize("rows", [500, 2])
@pytest.mark.parametrize("vocab", [8195, 40003])
@pytest.mark.parametrize("most", [0.0, 300.0, -1e3, 1e3, 1e4, -1e4, 1e5, 1e6, -1e6, 5e6, 8e6, -8e6])
def test_many_smaller_ones_first(most, vocab, rows):
    t = torch.arange(vocab, device="cuda", dtype=torch.float64)
    row = torch.where(t < vocab // 2, most - 6.0, torch.where(t % 97 == 5, most, most - 7.0))
    steps = most - 6.0 * (vocab - 1 - t).div(vocab // 5, rounding_mode="floor")
    logits = torch.stack([row, steps]).float().repeat(rows // 2, 1)
    check(logits, some_targets(rows, vocab, 3), 3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "f16", "f32"])
def test_behind_a_large_scale(dtype):
    t = torch.arange(20000, device="cuda")
    logits = torch.where(t < 10000, 29.0, torch.where(t % 97 == 5, 30.0, 28.75)).to(dtype).repeat(500, 1)
    for scale in (6.0, 7.0, 11.3, 24.0):
        check(logits, some_targets(500, 20000, 4), 3, scale)
        check(logits * 1000, some_targets(500, 20000, 4), 3, scale / 1000)
