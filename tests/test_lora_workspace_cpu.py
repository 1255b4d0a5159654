"""lora_add refuses a workspace whose elements do not follow one another (no GPU is needed: nothing is launched)."""
import pytest
import torch

from owoinfer_b200 import ops
from tests.test_text_ops_cpu import Plan, adapters, x


@pytest.mark.parametrize("workspace", [torch.zeros(1, dtype=torch.uint8).expand(4096), torch.zeros(8192, dtype=torch.uint8)[::2], torch.zeros(64, 64).t()], ids=["repeated", "strided", "turned"])
def test_refusals(workspace):
    with pytest.raises(ValueError, match="workspace"):
        ops.lora_add(torch.zeros(4, 128).bfloat16(), x, adapters(), Plan(), workspace=workspace)
