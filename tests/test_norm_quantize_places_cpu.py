"""add_rms_norm_quantize refuses outputs in the place of what other threads still read (no GPU is needed: nothing is launched)."""
import pytest

from owoinfer_b200 import _lib
from tests.test_text_ops_cpu import A, BF16, F16, F32, norm

B, D, E = A + (1 << 20), A + (2 << 20), A + (3 << 20)


@pytest.mark.parametrize("over,word", [
    (dict(residual_out=A, ld_residual_out=72, residual_dtype=BF16), "residual_out in"), (dict(residual_out=A, residual_dtype=F32), "residual_out in"),
    (dict(residual_out=B, ld_residual_out=68), "residual_out in"), (dict(x_dtype=F32, residual_out=A, ldx=68), "residual_out in"),
    (dict(norm_out=A, ld_norm=72), "norm_out in"), (dict(norm_out=A, x_dtype=F32), "norm_out in"), (dict(norm_out=E, residual_out=E, residual_dtype=BF16), "two matrices"),
    (dict(norm_out=A, residual_out=A, residual_dtype=BF16), "two matrices"), (dict(norm_out=A, norm_dtype=F16, ld_norm=72), "norm_out in"),
], ids=str)
def test_refusals(over, word):
    v = dict(tokens=2, x=A, residual=B, residual_out=B, norm_out=D, q=E + (1 << 20), scale=E + (2 << 20))
    v.update(over)
    assert norm(**v) == -1
    assert word in _lib.lib().b2_last_error_message().decode()
