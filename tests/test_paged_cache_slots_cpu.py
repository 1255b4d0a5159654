"""The largest block tables: a slot, and a stride of the kernels' loops behind it, is an int. (Addresses are never followed; no GPU is needed.)

Longest strides behind the last slot: the join of single-token attention takes 8 CTAs an SM 1024 slots further, eviction's threads look
up to 8192 slots past their share, a lane of the single-token kernel fetches entries of the block table 128 steps of 16 slots ahead. Past
2^31 they would turn negative, and pass for slots that exist."""
import pytest

from owoinfer_b200 import _lib
from tests.test_paged_cache_cpu import append, cache, decode, evict, prompt

MOST = 2 ** 31 - 2 ** 21


def wide(slots):
    return cache(page_size=1024, row_stride=128, head_stride=1024 * 128, page_stride=2 * 1024 * 128, table_width=slots // 1024, table_ld=slots // 1024)


def test_the_limit_covers_the_strides():
    sms = 160  # (of a whole GB100)
    assert MOST + max(8 * sms * 1024 + 4 * 256, 8192, 128 * 16) < 2 ** 31


@pytest.mark.parametrize("call", [append, prompt, decode, evict], ids=lambda f: f.__name__)
@pytest.mark.parametrize("slots", [MOST + 1024, 2 ** 31 - 1024])
def test_more_slots_are_refused(call, slots):
    assert call(c=wide(slots), **({"ld": 2 ** 31} if call is evict else {})) == -1
    assert "2^31 - 2^21" in _lib.lib().b2_last_error_message().decode()


def test_as_many_slots_are_taken():
    lib = _lib.lib()
    assert lib.b2_attention_paged_decode_workspace_bytes(wide(MOST), 4, 0, 0, 0, 1) > 256
    assert lib.b2_attention_paged_workspace_bytes(wide(MOST), 1, 4, 1, 0, 0) > 256
    assert lib.b2_attention_paged_decode_workspace_bytes(wide(MOST + 1024), 4, 0, 0, 0, 1) == 0
    assert lib.b2_attention_paged_workspace_bytes(wide(MOST + 1024), 1, 4, 1, 0, 0) == 0


def test_a_budget_past_the_limit_is_refused():
    assert evict(budget=MOST + 1, table_ld=2 ** 27, width=2 ** 27 - 1) == -1
    assert "2^31 - 2^21" in _lib.lib().b2_last_error_message().decode()
