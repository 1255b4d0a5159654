"""Matrices whose rows overlap (an expanded block table, say) have no row stride that the calls take: they are refused, not read past their end."""
import pytest
import torch

from owoinfer_b200 import ops


def pools():
    return torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16), torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16)


def table(rows, width):
    return torch.zeros((rows, width), dtype=torch.int32)


@pytest.mark.parametrize("width", [1, 4])
def test_an_expanded_block_table_is_refused(width):
    with pytest.raises(ValueError, match="block_table"):
        ops.PagedCache(*pools(), table(1, width).expand(3, width), torch.zeros(3, dtype=torch.int32))
    ops.PagedCache(*pools(), table(1, width).expand(3, width).contiguous(), torch.zeros(3, dtype=torch.int32))
    cache = ops.PagedCache(*pools(), table(1, 8)[:, :width].expand(1, width), torch.zeros(1, dtype=torch.int32))  # one row has no next one
    assert cache.struct.table_ld >= width
    assert ops.PagedCache(*pools(), table(3, 8)[:, :width], torch.zeros(3, dtype=torch.int32)).struct.table_ld == 8


def test_overlapping_rows_are_refused():
    cache = ops.PagedCache(*pools(), table(2, 4), torch.zeros(2, dtype=torch.int32))
    weights, cu = torch.zeros((2, 2, 64)), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="table_out"):
        ops.kv_evict(cache, weights, table(1, 1).expand(2, 1), 16)
    with pytest.raises(ValueError, match="table_out"):
        ops.kv_evict(cache, weights, table(1, 8)[0].as_strided((2, 4), (2, 1)), 16)
    row = torch.zeros((1, 8 * 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="qkv"):
        ops.qk_norm_rope_append(row.expand(5, 8 * 64), cache, cu, None, None, None)
