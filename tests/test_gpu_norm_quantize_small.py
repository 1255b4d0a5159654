"""add_rms_norm_quantize of rows so small that the norm's factor over the smallest scale passes 32 bits."""
import pytest
import torch

from owoinfer_b200 import ops
from tests.test_gpu_norm_quantize import check

pytestmark = pytest.mark.gpu
int8, e4m3 = torch.int8, torch.float8_e4m3fn


@pytest.mark.parametrize("codes", [int8, e4m3], ids=["int8", "e4m3"])
@pytest.mark.parametrize("group", [0, 32, 128])
@pytest.mark.parametrize("dim", [128, 4096])
@pytest.mark.parametrize("size", [1e-10, 1e-15])
def test_small_rows_without_an_eps(size, dim, group, codes):
    g = torch.Generator(device="cuda").manual_seed(dim)
    x = size * torch.randn(6, dim, generator=g, device="cuda")
    w = torch.ones(dim, device="cuda")
    x[1, :64] = 0.0                      # groups of zeros beside others that are not
    x[2, 32:64] *= 1e-29                 # a group whose scale is the smallest one (denormal numbers)
    x[3, 1:] = 0.0
    w[-32:] = 0.0                        # ... and one by its weights
    w[-64:-32] = 2.0 ** -70
    y = torch.empty(6, dim, dtype=torch.bfloat16, device="cuda")
    q, scale = ops.add_rms_norm_quantize(x, w, eps=0.0, dtype=codes, group=group, norm_out=y)
    check(x, None, w, codes, group, 0.0, q, scale, None, y, None)
    assert (q[1, :64].float() == 0).all() and (q[:, -32:].float() == 0).all()


@pytest.mark.parametrize("codes", [int8, e4m3], ids=["int8", "e4m3"])
@pytest.mark.parametrize("group", [0, 64])
@pytest.mark.parametrize("weight", [0.0, 1e-28, 1e-31, 1e-34])
def test_small_weights(weight, group, codes):
    g = torch.Generator(device="cuda").manual_seed(1)
    x = 1e-12 * torch.randn(3, 256, generator=g, device="cuda")
    w = torch.full((256,), weight, device="cuda")
    y = torch.empty(3, 256, dtype=torch.bfloat16, device="cuda")
    q, scale = ops.add_rms_norm_quantize(x, w, eps=0.0, dtype=codes, group=group, norm_out=y)
    # (1e-12 * 1e-28 and less are denormal, multiples of 2^-149 = 1.4e-45: only that the codes are in range is asked of them)
    if weight == 0.0:
        check(x, None, w, codes, group, 0.0, q, scale, None, y, None)
        assert (q.float() == 0).all()
    got = q.float()
    assert got.isfinite().all() and (got.sign() * x.sign() >= 0).all() and (scale >= 1e-30).all() and scale.isfinite().all()
