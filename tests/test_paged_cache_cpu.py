"""What the calls on paged key-value caches refuse, before any launch (no GPU is needed: addresses are never followed)."""
import ctypes as C

import pytest
import torch

from owoinfer_b200 import _lib, ops

A = 0x10000  # a 256-byte aligned address that nothing reads


def cache(**over):
    v = dict(struct_size=C.sizeof(_lib.PagedCache), k=A, v=A, page_stride=16 * 128 * 2, head_stride=16 * 128, row_stride=128, num_pages=10, dtype=0,
             kv_heads=2, page_size=16, head_dim=128, block_table=A, table_ld=4, table_width=4, seq_lens=A, batch=1)
    v.update(over)
    return _lib.PagedCache(*(v[name] for name, _ in _lib.PagedCache._fields_))


def view(tokens=1, heads=4, data=A, row=512, head=128):
    return _lib.View3(data, tokens, heads, row, head)


def append(c=None, qkv=A, ld=1024, tokens=1, q_heads=4, cu=A, q_norm=A, k_norm=A, eps=1e-6, rope=A, rows=8, rot=128, q_out=A, q_row=512, q_head=128):
    return _lib.lib().b2_qk_norm_rope_append(c or cache(), qkv, ld, tokens, q_heads, cu, None, q_norm, k_norm, eps, rope, rows, rot, 0, q_out, q_row, q_head, None)


def prompt(c=None, q=None, out=None, cu=A, max_q=1, scale=0.1, window=0, sinks=0, ws=A, ws_bytes=1 << 30):
    return _lib.lib().b2_attention_paged(c or cache(), q or view(), out or view(), None, cu, max_q, scale, window, sinks, ws, ws_bytes, None)


def decode(c=None, q=None, out=None, max_len=0, scale=0.1, window=0, sinks=0, weights=None, weights_out=None, ld=64, ws=A, ws_bytes=1 << 30):
    return _lib.lib().b2_attention_paged_decode(c or cache(), q or view(), out or view(), None, max_len, scale, window, sinks, weights, weights_out, ld, ws,
                                                ws_bytes, None)


def evict(c=None, weights=A, ld=64, sinks=0, recent=0, budget=16, table=A, table_ld=1, width=1, kept=A, lens=A, weights_out=None, out_ld=0):
    return _lib.lib().b2_kv_evict(c or cache(), weights, ld, sinks, recent, budget, table, table_ld, width, kept, lens, weights_out, out_ld, None)


BAD_CACHES = [
    (dict(struct_size=8), "struct_size"), (dict(dtype=2), "dtype"), (dict(head_dim=96), "head_dim"), (dict(page_size=8), "page_size"),
    (dict(page_size=48), "page_size"), (dict(page_size=2048), "page_size"), (dict(kv_heads=0), "kv_heads"), (dict(batch=-1), "batch"),
    (dict(batch=70000), "batch"), (dict(num_pages=-1), "num_pages"), (dict(table_width=1 << 28), "2^31"), (dict(table_ld=3), "table_ld"),
    (dict(row_stride=120), "row"), (dict(head_stride=2052), "strides"), (dict(page_stride=-8), "strides"), (dict(k=0), "pool"),
    (dict(v=A + 8), "aligned"), (dict(seq_lens=0), "seq_lens"), (dict(block_table=0), "block_table"),
]


@pytest.mark.parametrize("call", [append, prompt, decode, evict], ids=lambda f: f.__name__)
@pytest.mark.parametrize("over,word", BAD_CACHES, ids=[next(iter(o)) + str(next(iter(o.values()))) for o, _ in BAD_CACHES])
def test_bad_caches(call, over, word):
    assert call(c=cache(**over)) == -1
    assert word in _lib.lib().b2_last_error_message().decode()


@pytest.mark.parametrize("call,over,word", [
    (append, dict(tokens=-1), "tokens"), (append, dict(q_heads=0), "q_heads"), (append, dict(rot=24), "rot_dim"), (append, dict(rot=256), "rot_dim"),
    (append, dict(k_norm=None), "both or neither"), (append, dict(eps=-1.0), "eps"), (append, dict(eps=float("nan")), "eps"), (append, dict(cu=None), "cu_seqlens"),
    (append, dict(ld=1016), "qkv"), (append, dict(ld=1028), "qkv"), (append, dict(qkv=A + 2), "qkv"), (append, dict(q_out=None), "q_out"),
    (append, dict(q_head=4), "q_out"), (append, dict(rope=None), "rope"), (append, dict(rows=0), "rope"), (append, dict(q_norm=A + 4), "aligned"),
    (append, dict(c=cache(batch=0)), "without a sequence"),
    (prompt, dict(q=view(heads=3), out=view(heads=3)), "multiple of kv_heads"), (prompt, dict(out=view(tokens=2)), "same tokens"), (prompt, dict(scale=0.0), "scale"),
    (prompt, dict(scale=float("inf")), "scale"), (prompt, dict(window=-1), "window"), (prompt, dict(sinks=-1), "sinks"), (prompt, dict(max_q=-1), "max_q"),
    (prompt, dict(max_q=0), "max_q"), (prompt, dict(cu=None), "cu_seqlens"), (prompt, dict(q=view(data=A + 2)), "aligned"), (prompt, dict(out=view(row=516)), "multiples of 8"),
    (prompt, dict(c=cache(num_pages=0, k=0, v=0)), "no pages"),
    (prompt, dict(c=cache(table_width=4096, table_ld=4096), ws=None), "workspace"), (prompt, dict(c=cache(table_width=4096, table_ld=4096), ws=A + 16), "workspace"),
    (prompt, dict(c=cache(table_width=4096, table_ld=4096), ws_bytes=512), "workspace"),
    (decode, dict(q=view(tokens=2)), "one token"), (decode, dict(q=view(heads=5), out=view(heads=5)), "multiple of kv_heads"), (decode, dict(scale=-1.0), "scale"),
    (decode, dict(window=-2), "window"), (decode, dict(max_len=65), "max_len"), (decode, dict(max_len=-1), "max_len"), (decode, dict(weights=A), "both or neither"),
    (decode, dict(weights=A, weights_out=A, ld=63), "every slot"), (decode, dict(weights=A, weights_out=A, ws=None), "workspace"),
    (decode, dict(weights=A, weights_out=A, ws=A + 16), "workspace"), (decode, dict(weights=A, weights_out=A, ws_bytes=100), "workspace"),
    (decode, dict(q=view(data=None)), "aligned"),
    (evict, dict(budget=0), "budget"), (evict, dict(sinks=-1), "sinks"), (evict, dict(sinks=9, recent=8), "budget"), (evict, dict(width=0, table_ld=0), "table_out"),
    (evict, dict(table_ld=0), "table_out"), (evict, dict(ld=63), "weights"), (evict, dict(weights_out=A + 4096, out_ld=15), "weights_out"),
    (evict, dict(weights_out=A, out_ld=16), "weights_out"), (evict, dict(weights=None), "null"), (evict, dict(kept=None), "null"), (evict, dict(lens=None), "null"),
    (evict, dict(table=None), "null"),
])
def test_refusals(call, over, word):
    assert call(**over) == -1
    assert word in _lib.lib().b2_last_error_message().decode()


def test_nothing_to_do_launches_nothing():
    assert append(tokens=0) == 0
    assert prompt(q=view(tokens=0, data=None), out=view(tokens=0, data=None)) == 0
    empty = cache(batch=0, seq_lens=0, block_table=0)
    assert decode(c=empty, q=view(tokens=0, data=None), out=view(tokens=0, data=None)) == 0
    assert evict(c=empty) == 0
    assert _lib.lib().b2_paged_cache_status(None, 0) == -1


def test_workspace_sizes():
    size = lambda c, heads=4, max_len=0, window=0, weights=0: _lib.lib().b2_attention_paged_decode_workspace_bytes(c, heads, max_len, window, 0, weights)  # noqa: E731
    long = cache(table_width=4096, table_ld=4096)
    assert size(long, max_len=100000) == 0 and size(long, heads=5) == 0
    assert 0 < size(cache()) <= size(long, window=64) <= size(long) < size(long, weights=1)
    assert size(long, max_len=1000) < size(long) and size(long, max_len=1000, weights=1) < size(long, weights=1)


def test_workspace_sizes_of_prompts():
    size = lambda c, tokens=1, heads=4, max_q=1, window=0: _lib.lib().b2_attention_paged_workspace_bytes(c, tokens, heads, max_q, window, 0)  # noqa: E731
    long = cache(table_width=4096, table_ld=4096)
    assert size(cache()) == 256 and size(long, tokens=100000, max_q=100000) == 256  # nothing to cut, enough tokens
    assert size(long) > size(long, window=2000) > 256
    assert size(long, heads=5) == 0 and size(long, tokens=-1) == 0 and size(long, window=-1) == 0


def test_python_side_refusals():
    k = torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16)
    table, lens = torch.zeros((1, 4), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for args in ((k.float(), k.float(), table, lens), (k, k.half(), table, lens), (k, k[:, :1], table, lens), (k, k, table.long(), lens), (k, k, table, lens.long()),
                 (k, k, table, torch.zeros(2, dtype=torch.int32)), (k.transpose(2, 3), k.transpose(2, 3), table, lens), (k, k.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3), table, lens)):
        with pytest.raises(ValueError):
            ops.PagedCache(*args)
    c = ops.PagedCache(k, k.clone(), table, lens)
    q, cu = torch.zeros((1, 4, 64), dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    w = torch.zeros((1, 2, 64))
    for call in (lambda: ops.attention_paged(q.half(), c, cu, 1, 0.1), lambda: ops.attention_paged(q[..., :32], c, cu, 1, 0.1),
                 lambda: ops.attention_paged(q, c, torch.zeros(3, dtype=torch.int32), 1, 0.1), lambda: ops.attention_paged(q, c, cu, 1, 0.1, lse=torch.zeros(4)),
                 lambda: ops.attention_paged_decode(q, c, 0.1, weights=w[:, :1]), lambda: ops.attention_paged_decode(q, c, 0.1, weights=w, weights_out=w.double()),
                 lambda: ops.kv_evict(c, w.double(), table, 16), lambda: ops.kv_evict(c, w, table.long(), 16), lambda: ops.kv_evict(c, w, table, 0),
                 lambda: ops.kv_evict(c, w, table, 16, kept=torch.zeros((1, 2, 15), dtype=torch.int32)),
                 lambda: ops.qk_norm_rope_append(torch.zeros((1, 4 * 64), dtype=torch.bfloat16), c, cu, None, None, None),
                 lambda: ops.qk_norm_rope_append(torch.zeros((1, 8 * 64)), c, cu, None, None, None),
                 lambda: ops.qk_norm_rope_append(torch.zeros((1, 8 * 64), dtype=torch.bfloat16), c, cu, None, None, torch.zeros((4, 64), dtype=torch.bfloat16)),
                 lambda: ops.qk_norm_rope_append(torch.zeros((1, 8 * 64), dtype=torch.bfloat16), c, cu, torch.zeros(64), torch.zeros(64), None)):
        with pytest.raises(ValueError):
            call()
