"""Eviction reads the old lengths in every CTA while it writes the new ones: they are not the same buffer."""
import pytest
import torch

from owoinfer_b200 import _lib, ops
from tests.test_paged_cache_cpu import A, cache, evict


@pytest.mark.parametrize("lens", [A, A - 4, A + 8])
def test_lengths_in_place_are_refused(lens):
    assert evict(c=cache(batch=3), lens=lens) == -1
    assert "lens_out" in _lib.lib().b2_last_error_message().decode()


def test_lengths_in_place_are_refused_from_python(monkeypatch):
    monkeypatch.setattr(ops, "_raw_stream", lambda: 0)  # (there may be no GPU to ask)
    k, v = (torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16) for _ in range(2))
    table, lens = torch.zeros((1, 2), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="lens_out"):
        ops.kv_evict(ops.PagedCache(k, v, table, lens), torch.zeros((1, 2, 32)), table, 16, lens_out=lens)
