"""add_rms_norm_quantize of values half-way between two codes: to the even one, whatever the norm's factor."""
import pytest
import torch

from owoinfer_b200 import ops

pytestmark = pytest.mark.gpu
bf16 = torch.bfloat16


@pytest.mark.parametrize("group", [0, 256])
@pytest.mark.parametrize("dtype", [bf16, torch.float32], ids=["bf16", "f32"])
def test_half_way_between_integers(dtype, group):
    # s / max|s| * 127 is 0.5, 1.5, ... 126.5, 127 and their negatives in every row; the rows differ by powers of two (exact) and by an eps of their size.
    half = torch.cat([torch.arange(127, device="cuda") + 0.5, torch.tensor([127.0], device="cuda")])
    x = torch.cat([half, -half])
    x = (x * 2.0 ** torch.arange(-40, 40, device="cuda")[:, None]).to(dtype)
    assert torch.equal(x[40].float(), torch.cat([half, -half]))
    want = torch.round(torch.cat([half, -half])).to(torch.int8)
    for eps in (0.0, 1e-6, 0.3, 777.0):
        for rows in (x, x.repeat(30, 1), x[:, torch.randperm(256, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))].contiguous()):
            q, _ = ops.add_rms_norm_quantize(rows, eps=eps, group=group)
            order = torch.argsort(rows[-1].float())
            assert torch.equal(q[:, order], want[torch.argsort(torch.cat([half, -half]))].expand(len(rows), -1))


@pytest.mark.parametrize("group", [0, 128])
def test_half_way_between_e4m3(group):
    # Between neighbouring codes from 16 to 448, of rows whose largest is 448 times a power of two.
    codes = torch.arange(256, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn).float()
    codes = torch.sort(codes[codes.isfinite() & (codes >= 16)])[0]
    border = ((codes[1:] + codes[:-1]) / 2)
    row = torch.cat([border, codes[-1:], torch.zeros(128 - len(border) - 1, device="cuda")])
    x = row * 2.0 ** torch.arange(-40, 40, device="cuda")[:, None]
    want = row.double()
    step = torch.exp2(torch.floor(torch.log2(want.clamp(min=2.0 ** -6))) - 3)
    want = torch.round(want / step) * step
    for eps in (0.0, 1e-6, 0.3, 777.0):
        for k in (1, 20):
            q, _ = ops.add_rms_norm_quantize(x.repeat(k, 1), eps=eps, dtype=torch.float8_e4m3fn, group=group)
            assert torch.equal(q.double(), want.expand(80 * k, -1))
