"""lora_add in half precision: an infinity in x A^T beside numbers past the type's own largest."""
import pytest
import torch

from owoinfer_b200 import ops

pytestmark = pytest.mark.gpu


# (each of the ways that a call can go)
@pytest.mark.parametrize("tokens,rank,adapters", [(40, 8, 2), (70, 32, 2), (1300, 16, 2), (17000, 16, 2), (1600, 64, 2), (1100, 128, 40)])
def test_an_infinity_beside_large_numbers(tokens, rank, adapters):
    g = torch.Generator(device="cuda").manual_seed(rank)
    x = torch.ones(tokens, 64, device="cuda").half()
    a, b = torch.zeros(adapters, rank, 64, device="cuda").half(), torch.zeros(adapters, 24, rank, device="cuda").half()
    a[:, 0, 0] = float("inf")
    a[:, 1:5, :] = 3000.0  # sums of 192000, past fp16's 65504
    b[:, :, 0] = torch.where(torch.rand(24, generator=g, device="cuda") < 0.5, -1.0, 1.0).half()
    b[:, :, 1:5] = -b[:, :, :1]
    y = torch.randn(tokens, 24, generator=g, device="cuda").half()
    ids = torch.arange(tokens, dtype=torch.int32, device="cuda") % adapters
    got = ops.lora_add(y, x, ops.LoraAdapters(a, b), ops.LoraPlan(ids, adapters), out=torch.empty_like(y))
    # inf b_0 + 4 * 192000 (-b_0): the infinity, of b_0's sign
    assert torch.equal(got.float(), b[ids.long(), :, 0].float() * float("inf"))
