"""The rank that token_logprobs gives a target of plus infinity: what equals it counts only ahead of it."""
import math

import pytest
import torch

from tests.test_gpu_logprobs import check, rows_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,vocab", [(1000, 8192), (1000, 16384), (300, 70001), (40, 50), (2, 64007)])
def test_equal_infinities(rows, vocab, dtype):
    logits = rows_of(rows, vocab, dtype, seed=4).contiguous()
    row = torch.arange(rows, device="cuda")
    first = row * 13 % (vocab // 2)
    for apart in (1, 9, 300, 4096, vocab // 2):
        second = (first + apart).clamp(max=vocab - 1)
        some = logits.clone()
        some[row, first] = some[row, second] = math.inf
        check(some, first, 3)
        check(some, second, 3)
    some[:, ::7] = math.inf
    check(some, row % vocab // 7 * 7, 3)
