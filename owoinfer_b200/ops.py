"""Host-side mirror of the reference's kernel-level interface for the quantized DiT block, over torch CUDA tensors.

Same names, argument meaning and error behaviour as the reference's C++ entry points (kernels::quant::*,
kernels::quant4::*, attention_q8::attention_q8, kernels::fused::qk_norm_rope_moss, moss_dit::run_block_quant); every
function calls straight into the C ABI of libowoinfer_b200.so on the current torch stream. torch is used for device
memory and streams only. Invalid arguments raise ValueError (the reference throws std::invalid_argument).
"""
from __future__ import annotations

import ctypes as C
import functools
import math
import typing

import torch

from . import _lib
from ._lib import check

TILE_AUTO, TILE_128x256, TILE_128x128, TILE_2CTA_256x256 = 0, 1, 2, 3
TIER_INT8, TIER_W4A4_VIA_INT8, TIER_W4A8 = 0, 1, 2
ATTENTION_Q8_FP8 = 2          # e4m3 P.V with the ranges of the fp16-accumulating variant (112 / 4.5); accumulated in fp32 here
ATTENTION_Q8_FP8_F32ACC = 3


def _stream() -> C.c_void_p:
    if not torch.cuda.is_initialized():
        return C.c_void_p(torch.cuda.current_stream().cuda_stream)
    # The same handle without the Stream object around it, whose making is a good part of a small call.
    try:
        return C.c_void_p(torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice()))
    except AttributeError:  # private names, which another torch may not have
        return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _ptr(t) -> C.c_void_p:
    return C.c_void_p(0 if t is None else t.data_ptr())


def _ld(t) -> int:
    return t.stride(0) if t.dim() == 2 and t.shape[0] > 1 else t.shape[-1]


# ------------------------------------------------------------------------------------------------ quantisers

def rotate_quantize(x, q=None, scale=None):
    m, k = x.shape
    q = torch.empty((m, k), dtype=torch.int8, device=x.device) if q is None else q
    scale = torch.empty(m, dtype=torch.float32, device=x.device) if scale is None else scale
    check(_lib.lib().b2_rotate_quantize(_ptr(x), C.c_int64(_ld(x)), _ptr(q), C.c_int64(_ld(q)), _ptr(scale), C.c_int64(m),
                                        C.c_int(k), _stream()))
    return q, scale


def rms_norm_modulate_rotate_quantize(x, norm_weight, mod_scale, mod_shift, q=None, scale=None, y=None):
    m, k = x.shape
    q = torch.empty((m, k), dtype=torch.int8, device=x.device) if q is None else q
    scale = torch.empty(m, dtype=torch.float32, device=x.device) if scale is None else scale
    check(_lib.lib().b2_rms_norm_modulate_rotate_quantize(
        _ptr(x), C.c_int64(_ld(x)), _ptr(norm_weight), _ptr(mod_scale), _ptr(mod_shift), _ptr(q), C.c_int64(_ld(q)),
        _ptr(scale), C.c_int64(m), C.c_int(k), _stream(), _ptr(y), C.c_int64(0 if y is None else _ld(y))))
    return q, scale


def convrot_quantize_int4(x, q=None, scale=None):
    m, k = x.shape
    q = torch.empty((m, k // 2), dtype=torch.uint8, device=x.device) if q is None else q
    scale = torch.empty(m, dtype=torch.float32, device=x.device) if scale is None else scale
    check(_lib.lib().b2_convrot_quantize_int4(_ptr(x), C.c_int64(_ld(x)), _ptr(q), C.c_int64(_ld(q)), _ptr(scale),
                                              C.c_int64(m), C.c_int(k), _stream()))
    return q, scale


def rms_norm_modulate_convrot_quantize_int4(x, norm_weight, mod_scale, mod_shift, q=None, scale=None):
    m, k = x.shape
    q = torch.empty((m, k // 2), dtype=torch.uint8, device=x.device) if q is None else q
    scale = torch.empty(m, dtype=torch.float32, device=x.device) if scale is None else scale
    check(_lib.lib().b2_rms_norm_modulate_convrot_quantize_int4(
        _ptr(x), C.c_int64(_ld(x)), _ptr(norm_weight), _ptr(mod_scale), _ptr(mod_shift), _ptr(q), C.c_int64(_ld(q)),
        _ptr(scale), C.c_int64(m), C.c_int(k), _stream()))
    return q, scale


def unpack_int4(packed, out=None):
    rows, kb = packed.shape
    out = torch.empty((rows, kb * 2), dtype=torch.int8, device=packed.device) if out is None else out
    check(_lib.lib().b2_unpack_int4(_ptr(packed), C.c_int64(_ld(packed)), _ptr(out), C.c_int64(_ld(out)), C.c_int64(rows),
                                    C.c_int64(kb * 2), _stream()))
    return out


def decode_grouped_int8(packed, s_rel, group, codebook=None, out=None, invalid=None):
    """invalid: optional uint32/int32 device tensor of one element, OR-ed with 1 when a group scale is NaN or negative."""
    rows, kb = packed.shape
    k = kb * 2
    kind = 0 if s_rel.dtype in (torch.uint8, torch.int8) else 1
    out = torch.empty((rows, k), dtype=torch.int8, device=packed.device) if out is None else out
    check(_lib.lib().b2_decode_grouped_int8(_ptr(packed), _ptr(s_rel), C.c_int(kind), _ptr(codebook), C.c_int64(rows),
                                            C.c_int64(k), C.c_int(group), _ptr(out), _ptr(invalid), _stream()))
    return out


def w4_invalid_scales(clear=False):
    v = C.c_uint(0)
    check(_lib.lib().b2_w4_invalid_scales(C.byref(v), C.c_int(1 if clear else 0)))
    return int(v.value)


# ------------------------------------------------------------------------------------------------ GEMMs

def _operands(x_q, x_scale, w, w_scale):
    m, k = x_q.shape
    return _lib.Int8Operands(x_q.data_ptr(), _ld(x_q), x_scale.data_ptr(), w.data_ptr(), w_scale.data_ptr(), m, w.shape[0], k)


def int8_gemm(x_q, x_scale, w, w_scale, bias=None, out=None, tile=TILE_AUTO):
    op = _operands(x_q, x_scale, w, w_scale)
    out = torch.empty((op.m, op.n), dtype=torch.bfloat16, device=x_q.device) if out is None else out
    check(_lib.lib().b2_int8_gemm(C.byref(op), _ptr(bias), _ptr(out), C.c_int64(_ld(out)), _stream(), C.c_int(tile)))
    return out


def int8_gemm_chunked(x_q, x_scale, w, w_scale, chunk_cols, bias=None, out=None, tile=TILE_AUTO):
    """The plain GEMM with its output split by columns: out is [n / chunk_cols, m, chunk_cols]."""
    op = _operands(x_q, x_scale, w, w_scale)
    chunks = op.n // chunk_cols
    out = torch.empty((chunks, op.m, chunk_cols), dtype=torch.bfloat16, device=x_q.device) if out is None else out
    check(_lib.lib().b2_int8_gemm_chunked(C.byref(op), _ptr(bias), _ptr(out), C.c_int64(out.stride(1)), C.c_int(chunk_cols),
                                          C.c_int64(out.stride(0)), _stream(), C.c_int(tile)))
    return out


def rotate_quantize_chunked(x_chunks, q=None, scale=None):
    """x_chunks: bf16 [chunks, m, chunk_cols]; quantises the rows of the column-concatenated [m, chunks * chunk_cols]."""
    chunks, m, cw = x_chunks.shape
    k = chunks * cw
    q = torch.empty((m, k), dtype=torch.int8, device=x_chunks.device) if q is None else q
    scale = torch.empty(m, dtype=torch.float32, device=x_chunks.device) if scale is None else scale
    check(_lib.lib().b2_rotate_quantize_chunked(_ptr(x_chunks), C.c_int64(x_chunks.stride(1)), C.c_int(cw),
                                                C.c_int64(x_chunks.stride(0)), _ptr(q), C.c_int64(_ld(q)), _ptr(scale),
                                                C.c_int64(m), C.c_int(k), _stream()))
    return q, scale


def int8_gemm_gated_residual(x_q, x_scale, w, w_scale, gate, residual, bias=None, tile=TILE_AUTO):
    op = _operands(x_q, x_scale, w, w_scale)
    check(_lib.lib().b2_int8_gemm_gated_residual(C.byref(op), _ptr(bias), _ptr(gate), _ptr(residual),
                                                 C.c_int64(_ld(residual)), _stream(), C.c_int(tile)))
    return residual


def int8_gemm_situ_glu(x_q, x_scale, w, w_scale, out=None, tile=TILE_AUTO):
    op = _operands(x_q, x_scale, w, w_scale)
    out = torch.empty((op.m, op.n // 2), dtype=torch.bfloat16, device=x_q.device) if out is None else out
    check(_lib.lib().b2_int8_gemm_situ_glu(C.byref(op), _ptr(out), C.c_int64(_ld(out)), _stream(), C.c_int(tile)))
    return out


def int8_gemm_acc(x_q, w, tile=TILE_AUTO):
    m, k = x_q.shape
    ones = torch.ones(max(m, w.shape[0], 4), dtype=torch.float32, device=x_q.device)
    op = _operands(x_q, ones, w, ones)
    acc = torch.empty((m, w.shape[0]), dtype=torch.int32, device=x_q.device)
    check(_lib.lib().b2_int8_gemm_acc(C.byref(op), _ptr(acc), C.c_int64(w.shape[0]), _stream(), C.c_int(tile)))
    return acc


def make_w4(packed, s_rel, group, s_channel, codebook=None):
    kind = 0 if s_rel.dtype in (torch.uint8, torch.int8) else 1
    w = _lib.W4Weight(packed.data_ptr(), s_rel.data_ptr(), kind, group, 0 if codebook is None else codebook.data_ptr(),
                      s_channel.data_ptr())
    w._keep = (packed, s_rel, s_channel, codebook)
    return w


def debug_w4a8_route(route: int):
    """-1 automatic, 0 always decode to the scratch, 1 decode inside the GEMM whenever the weight's format allows."""
    check(_lib.lib().b2_debug_w4a8_route(C.c_int(route)))


def w4a8_gemm(x_q, x_scale, w4, n, epilogue=0, aux=None, out=None, scratch=None):
    """scratch: int8 [n, k] for the weights that are decoded ahead of the GEMM (allocated when None); False passes no
    scratch at all (only weights the fused kernel takes: e4m3 scales, tile-sized shapes)."""
    m, k = x_q.shape
    if scratch is False:
        scratch = None
    elif scratch is None:
        scratch = torch.empty((n, k), dtype=torch.int8, device=x_q.device)
    if out is None:
        out = torch.empty((m, n // 2 if epilogue == 2 else n), dtype=torch.bfloat16, device=x_q.device)
    check(_lib.lib().b2_w4a8_gemm(_ptr(x_q), C.c_int64(_ld(x_q)), _ptr(x_scale), C.byref(w4), C.c_int64(m), C.c_int64(n),
                                  C.c_int64(k), C.c_int(epilogue), _ptr(aux), _ptr(out), C.c_int64(_ld(out)),
                                  _ptr(scratch), _stream()))
    return out


# ------------------------------------------------------------------------------------------------ attention side

def qk_norm_rope_moss(qkv, heads, q_norm, k_norm, table):
    check(_lib.lib().b2_qk_norm_rope_moss(_ptr(qkv), C.c_int64(_ld(qkv)), C.c_int64(qkv.shape[0]), C.c_int(heads),
                                          _ptr(q_norm), _ptr(k_norm), _ptr(table), C.c_int64(_ld(table)), _stream()))
    return qkv


def moss_rope_table(height, width, text_length, device="cuda"):
    n = height * width + text_length
    out = torch.empty((n, 128), dtype=torch.bfloat16, device=device)
    check(_lib.lib().b2_moss_rope_table(_ptr(out), C.c_int64(128), C.c_int(height), C.c_int(width), C.c_int(text_length),
                                        _stream()))
    return out


def moss_rope_table_reference(height, width, index, device="cuda"):
    out = torch.empty((height * width, 128), dtype=torch.bfloat16, device=device)
    check(_lib.lib().b2_moss_rope_table_reference(_ptr(out), C.c_int64(128), C.c_int(height), C.c_int(width), C.c_int(index),
                                                  _stream()))
    return out


def _view3(t):
    return _lib.View3(t.data_ptr(), t.shape[0], t.shape[1], t.stride(0), t.stride(1))


def attention_options(p_range=0.0, v_range=0.0, variant=ATTENTION_Q8_FP8_F32ACC):
    return _lib.AttentionOptions(variant, p_range, v_range)


def attention_q8_workspace_bytes(total_q, total_k, batch, max_seqlen, heads, kv_heads=None, options=None):
    o = options or attention_options()
    return int(_lib.lib().b2_attention_q8_workspace_bytes(C.byref(o), total_q, total_k, batch, max_seqlen, heads,
                                                          heads if kv_heads is None else kv_heads))


def attention_q8_layout(total_q, total_k, batch, max_seqlen, heads, options=None):
    o = options or attention_options()
    l = _lib.AttentionLayout()
    check(_lib.lib().b2_attention_q8_layout(C.byref(o), C.c_int64(total_q), C.c_int64(total_k), C.c_int(batch),
                                            C.c_int(max_seqlen), C.c_int(heads), C.c_int(heads), C.byref(l)))
    return l


def attention_q8(q, k, v, out, cu_seqlens_q, cu_seqlens_k, max_seqlen, scale, workspace=None, options=None,
                 norm_rope=None):
    """q, k, v, out: bf16 [tokens, heads, 128] views (head_dim contiguous). norm_rope: (q_norm, k_norm, table) or None."""
    o = options or attention_options()
    batch = cu_seqlens_q.shape[0] - 1
    if workspace is None:
        nbytes = attention_q8_workspace_bytes(q.shape[0], k.shape[0], batch, max_seqlen, q.shape[1], k.shape[1], o)
        workspace = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=q.device)
    nr = None
    if norm_rope is not None:
        nr = _lib.QkNormRope(norm_rope[0].data_ptr(), norm_rope[1].data_ptr(), norm_rope[2].data_ptr(), _ld(norm_rope[2]))
    vq, vk, vv, vo = _view3(q), _view3(k), _view3(v), _view3(out)
    check(_lib.lib().b2_attention_q8(C.byref(o), C.byref(vq), C.byref(vk), C.byref(vv), C.byref(vo), _ptr(cu_seqlens_q),
                                     _ptr(cu_seqlens_k), C.c_int(batch), C.c_int(max_seqlen), C.c_float(scale),
                                     _ptr(workspace), C.c_size_t(workspace.numel()), _stream(),
                                     None if nr is None else C.byref(nr)))
    return out, workspace


def attention_q8_preprocess(q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen, workspace=None, options=None, norm_rope=None):
    """The pre-pass of attention_q8 alone; returns the workspace it filled."""
    o = options or attention_options()
    batch = cu_seqlens_q.shape[0] - 1
    if workspace is None:
        nbytes = attention_q8_workspace_bytes(q.shape[0], k.shape[0], batch, max_seqlen, q.shape[1], k.shape[1], o)
        workspace = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=q.device)
    nr = None
    if norm_rope is not None:
        nr = _lib.QkNormRope(norm_rope[0].data_ptr(), norm_rope[1].data_ptr(), norm_rope[2].data_ptr(), _ld(norm_rope[2]))
    vq, vk, vv = _view3(q), _view3(k), _view3(v)
    check(_lib.lib().b2_attention_q8_preprocess(C.byref(o), C.byref(vq), C.byref(vk), C.byref(vv), _ptr(cu_seqlens_q),
                                                _ptr(cu_seqlens_k), C.c_int(batch), C.c_int(max_seqlen), _ptr(workspace),
                                                C.c_size_t(workspace.numel()), _stream(), None if nr is None else C.byref(nr)))
    return workspace


def attention_q8_debug_scores(q, k, v, out, cu_seqlens_q, cu_seqlens_k, max_seqlen, scale, seq, head, tile_q, workspace=None,
                              options=None, norm_rope=None):
    """attention_q8 that also returns the attention kernel's own int32 Q·K^T accumulators of one (sequence, head, 128-row
    query tile): (int32 [128, 64 * ceil(max_seqlen / 64)], workspace)."""
    o = options or attention_options()
    batch = cu_seqlens_q.shape[0] - 1
    if workspace is None:
        nbytes = attention_q8_workspace_bytes(q.shape[0], k.shape[0], batch, max_seqlen, q.shape[1], k.shape[1], o)
        workspace = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=q.device)
    nr = None
    if norm_rope is not None:
        nr = _lib.QkNormRope(norm_rope[0].data_ptr(), norm_rope[1].data_ptr(), norm_rope[2].data_ptr(), _ld(norm_rope[2]))
    ld = (max_seqlen + 63) // 64 * 64
    scores = torch.zeros((128, ld), dtype=torch.int32, device=q.device)
    vq, vk, vv, vo = _view3(q), _view3(k), _view3(v), _view3(out)
    check(_lib.lib().b2_attention_q8_debug_scores(C.byref(o), C.byref(vq), C.byref(vk), C.byref(vv), C.byref(vo),
                                                  _ptr(cu_seqlens_q), _ptr(cu_seqlens_k), C.c_int(batch), C.c_int(max_seqlen),
                                                  C.c_float(scale), _ptr(workspace), C.c_size_t(workspace.numel()), _stream(),
                                                  None if nr is None else C.byref(nr), C.c_int(seq), C.c_int(head),
                                                  C.c_int(tile_q), _ptr(scores), C.c_int64(ld)))
    return scores, workspace


def kernel_status():
    g, a = C.c_int(0), C.c_int(0)
    check(_lib.lib().b2_kernel_status(C.byref(g), C.byref(a)))
    return g.value, a.value


def kernel_status_clear():
    check(_lib.lib().b2_kernel_status_clear())


def debug_bounded_wait(wait_limit_ns: int, skip_gemm_stage: int):
    check(_lib.lib().b2_debug_bounded_wait(C.c_uint64(wait_limit_ns), C.c_int(int(skip_gemm_stage))))


# ------------------------------------------------------------------------------------------------ block / step

class BlockWeights:
    """Device weights of one all-quantized block (BlockTensors of the reference, restricted to this route).

    qkv / o / up_gate / down: (int8 weight [n, k], f32 scale [n]) for TIER_INT8; (packed int4 uint8 [n, k/2], f32 scale)
    for TIER_W4A4_VIA_INT8; a W4Weight from make_w4 for TIER_W4A8.
    """

    def __init__(self, norm1, norm2, q_norm, k_norm, qkv, o, up_gate, down):
        self.tensors = (norm1, norm2, q_norm, k_norm, qkv, o, up_gate, down)
        s = _lib.BlockWeights()
        s.struct_size = C.sizeof(_lib.BlockWeights)
        s.norm1, s.norm2, s.q_norm, s.k_norm = (t.data_ptr() for t in (norm1, norm2, q_norm, k_norm))
        for name, lin in (("qkv", qkv), ("o", o), ("up_gate", up_gate), ("down", down)):
            l = _lib.Linear()
            if isinstance(lin, _lib.W4Weight):
                l.w4 = C.pointer(lin)
            else:
                l.w, l.scale = lin[0].data_ptr(), lin[1].data_ptr()
            setattr(s, name, l)
        self.struct = s


def block_run(tokens, cu_seqlens, max_seqlen, D=3072, F=12288, heads=24, tier=TIER_INT8, p_range=0.0, v_range=0.0,
              fused_norm_rope=-1, slot_rows=0, slot_kv=(None, None), cu_seqlens_k=None, k0=0, k1=0, kv_tap=None, tap_only=False,
              slot_kv_ld=0, attention_variant=ATTENTION_Q8_FP8_F32ACC):
    r = _lib.BlockRun()
    r.struct_size = C.sizeof(_lib.BlockRun)
    r.tokens, r.D, r.F, r.heads = tokens, D, F, heads
    r.cu_seqlens = cu_seqlens.data_ptr()
    r.batch, r.max_seqlen, r.tier = cu_seqlens.shape[0] - 1, max_seqlen, tier
    r.attention = attention_options(p_range, v_range, attention_variant)
    r.fused_norm_rope = fused_norm_rope
    r.slot_rows, r.k0, r.k1, r.tap_only, r.slot_kv_ld = slot_rows, k0, k1, int(tap_only), slot_kv_ld
    r.slot_kv[0], r.slot_kv[1] = (None if t is None else t.data_ptr() for t in slot_kv)
    r.cu_seqlens_k = None if cu_seqlens_k is None else cu_seqlens_k.data_ptr()
    r.kv_tap = None if kv_tap is None else kv_tap.data_ptr()
    r._keep = (cu_seqlens, slot_kv, cu_seqlens_k, kv_tap)
    return r


def block_quant_workspace_bytes(run) -> int:
    n = int(_lib.lib().b2_block_quant_workspace_bytes(C.byref(run)))
    if n == 0:
        raise ValueError(_lib.lib().b2_last_error_message().decode())
    return n


def block_buffers(x, mod, rope, workspace):
    b = _lib.BlockBuffers()
    b.struct_size = C.sizeof(_lib.BlockBuffers)
    b.x, b.mod, b.rope, b.workspace, b.workspace_bytes = x.data_ptr(), mod.data_ptr(), rope.data_ptr(), workspace.data_ptr(), workspace.numel()
    b._keep = (x, mod, rope, workspace)
    return b


def run_block_quant(weights: BlockWeights, buffers, run):
    check(_lib.lib().b2_run_block_quant(C.byref(weights.struct), C.byref(buffers), C.byref(run), _stream()))


def dit_step(blocks, buffers, run):
    arr = (_lib.BlockWeights * len(blocks))(*[b.struct for b in blocks])
    check(_lib.lib().b2_dit_step(arr, C.c_int(len(blocks)), C.byref(buffers), C.byref(run), _stream()))


SM_SCALE = 1.0 / math.sqrt(128.0)


# ------------------------------------------------------------------------------------------------ sequence parallel

class SpComm:
    """Communicator of one sequence-parallel group (b2_sp_comm). `unique_id` is the bytes rank 0 of the group got from
    sp_unique_id(); size 1 needs none."""

    def __init__(self, size: int, rank: int, unique_id: bytes | None = None):
        self.size, self.rank = size, rank
        self.handle = C.c_void_p()
        buf = (C.c_char * 128).from_buffer_copy(unique_id) if unique_id is not None else None
        check(_lib.lib().b2_sp_comm_create(buf, C.c_size_t(128 if buf is not None else 0), C.c_int(size), C.c_int(rank),
                                           C.byref(self.handle)))

    def local_exchange(self, on: bool):
        check(_lib.lib().b2_sp_comm_local_exchange(self.handle, C.c_int(1 if on else 0)))

    def close(self):
        if self.handle:
            _lib.lib().b2_sp_comm_destroy(self.handle)
            self.handle = C.c_void_p()


def sp_unique_id() -> bytes:
    buf = (C.c_char * 128)()
    check(_lib.lib().b2_sp_unique_id(buf, C.c_size_t(128)))
    return bytes(buf)


def sp_run(seq_lens, size, cu_seqlens_full, D=3072, F=12288, heads=24, fused_norm_rope=-1):
    """b2_sp_run of one rank: seq_lens are the FULL sequence lengths (host ints), cu_seqlens_full their device prefix sums."""
    r = _lib.SpRun()
    r.struct_size = C.sizeof(_lib.SpRun)
    r.local = block_run(sum(s // size for s in seq_lens), cu_seqlens_full, max(seq_lens), D=D, F=F, heads=heads,
                        fused_norm_rope=fused_norm_rope)
    arr = (C.c_int32 * len(seq_lens))(*seq_lens)
    r.seq_lens_host = C.cast(arr, C.c_void_p)
    r._keep = (arr, cu_seqlens_full)
    return r


def block_quant_sp_workspace_bytes(run, size) -> int:
    n = int(_lib.lib().b2_block_quant_sp_workspace_bytes(C.byref(run), C.c_int(size)))
    if n == 0:
        raise ValueError(_lib.lib().b2_last_error_message().decode())
    return n


def run_block_quant_sp(weights: BlockWeights, bufs, run, comm: SpComm):
    check(_lib.lib().b2_run_block_quant_sp(C.byref(weights.struct), C.byref(bufs), C.byref(run), comm.handle, _stream()))


def dit_step_sp(blocks, bufs, run, comm: SpComm):
    arr = (_lib.BlockWeights * len(blocks))(*[b.struct for b in blocks])
    check(_lib.lib().b2_dit_step_sp(arr, C.c_int(len(blocks)), C.byref(bufs), C.byref(run), comm.handle, _stream()))


# ------------------------------------------------------------------------------------------------ guidance + update

def cfg_combine(cond, uncond, g, out=None):
    out = torch.empty_like(cond) if out is None else out
    check(_lib.lib().b2_cfg_combine(_ptr(cond), _ptr(uncond), C.c_float(g), _ptr(out), C.c_int64(cond.numel()), _stream()))
    return out


def slg_correct(pred, cond, skipped, scale, out=None):
    out = torch.empty_like(cond) if out is None else out
    check(_lib.lib().b2_slg_correct(_ptr(pred), _ptr(cond), _ptr(skipped), C.c_float(scale), _ptr(out), C.c_int64(cond.numel()),
                                    _stream()))
    return out


def euler_update(x, v, h):
    check(_lib.lib().b2_euler_update(_ptr(x), _ptr(v), C.c_float(h), C.c_int64(x.numel()), _stream()))
    return x


def ab2_update(x, v, v_prev, h, a, b):
    check(_lib.lib().b2_ab2_update(_ptr(x), _ptr(v), _ptr(v_prev), C.c_float(h), C.c_float(a), C.c_float(b), C.c_int64(x.numel()),
                                   _stream()))
    return x


def guided_velocity_step(v_cond, x=None, v_uncond=None, v_skip=None, v_prev=None, v_out=None, cfg_scale=0.0, slg_scale=0.0,
                         h=0.0, a=0.0, b=0.0, update=0):
    """One pass: guidance (cfg when v_uncond is given, slg when v_skip is given), optional store of the guided velocity,
    and the Euler (update 1) or Adams-Bashforth (update 2) step of x."""
    # (Filled in one go: the kernel is a microsecond or two, so the host's side of this call is most of its time.)
    g = _lib.GuidedStep(C.sizeof(_lib.GuidedStep), None if x is None else x.data_ptr(), None if v_cond is None else v_cond.data_ptr(),
                        None if v_uncond is None else v_uncond.data_ptr(), None if v_skip is None else v_skip.data_ptr(),
                        None if v_prev is None else v_prev.data_ptr(), None if v_out is None else v_out.data_ptr(), cfg_scale, slg_scale,
                        h, a, b, int(v_uncond is not None), int(v_skip is not None), update, v_cond.numel())
    check(_lib.lib().b2_guided_velocity_step(C.byref(g), _stream()))
    return x if update else v_out


# ------------------------------------------------------------------------------------------------ forward shell

def latent_to_tokens(latents, tokens=None, col0=0):
    """f32 [C, h, w] (or [C, hw]) -> bf16 [hw, C]; into columns [col0, col0 + C) of a wider `tokens` when given."""
    c, hw = latents.shape[0], latents.numel() // latents.shape[0]
    tokens = torch.empty((hw, c), dtype=torch.bfloat16, device=latents.device) if tokens is None else tokens
    dst = C.c_void_p(tokens.data_ptr() + 2 * col0)
    check(_lib.lib().b2_latent_to_tokens(_ptr(latents), C.c_int(c), C.c_int64(hw), dst, C.c_int64(tokens.stride(0)), _stream()))
    return tokens


def tokens_to_latent(tokens, latents=None):
    hw, c = tokens.shape
    latents = torch.empty((c, hw), dtype=torch.float32, device=tokens.device) if latents is None else latents
    check(_lib.lib().b2_tokens_to_latent(_ptr(tokens), _ptr(latents), C.c_int(c), C.c_int64(hw), _stream()))
    return latents


def linear_fp32_row(w, x, bias, out=None):
    n, k = w.shape
    out = torch.empty(n, dtype=torch.bfloat16, device=w.device) if out is None else out
    check(_lib.lib().b2_linear_fp32_row(_ptr(w), _ptr(x), _ptr(bias), _ptr(out), C.c_int(n), C.c_int(k), _stream()))
    return out


def rms_norm_modulate(x, norm_weight, mod_scale, mod_shift, y=None):
    m, k = x.shape
    y = torch.empty((m, k), dtype=torch.bfloat16, device=x.device) if y is None else y
    check(_lib.lib().b2_rms_norm_modulate(_ptr(x), C.c_int64(_ld(x)), _ptr(norm_weight), _ptr(mod_scale), _ptr(mod_shift),
                                          _ptr(y), C.c_int64(_ld(y)), C.c_int64(m), C.c_int(k), _stream()))
    return y


def time_sinusoid(timestep):
    import numpy as np
    emb = np.empty(256, np.float32)
    check(_lib.lib().b2_time_sinusoid(C.c_float(timestep), emb.ctypes.data_as(C.c_void_p)))
    return emb


def time_vector_fp32(w0, b0, w2, b2, timestep):
    """Host: numpy f32 weights of the timestep MLP -> the f32 time vector [dim]."""
    import numpy as np
    w0, b0, w2, b2 = (np.ascontiguousarray(a, np.float32) for a in (w0, b0, w2, b2))
    te = _lib.TimeEmbedding()
    te.struct_size, te.dim = C.sizeof(_lib.TimeEmbedding), w2.shape[0]
    te.w0, te.b0, te.w2, te.b2 = (a.ctypes.data for a in (w0, b0, w2, b2))
    out = np.empty(w2.shape[0], np.float32)
    check(_lib.lib().b2_time_vector_fp32(C.byref(te), C.c_float(timestep), out.ctypes.data_as(C.c_void_p)))
    return out


def linear_bf16(x, w, bias=None, out=None, workspace=None):
    m, k = x.shape
    n = w.shape[0]
    out = torch.empty((m, n), dtype=torch.bfloat16, device=x.device) if out is None else out
    if workspace is None:
        workspace = torch.empty(_lib.lib().b2_linear_bf16_workspace_bytes(), dtype=torch.uint8, device=x.device)
    check(_lib.lib().b2_linear_bf16(_ptr(x), C.c_int64(_ld(x)), _ptr(w), _ptr(bias), _ptr(out), C.c_int64(_ld(out)),
                                    C.c_int64(m), C.c_int(n), C.c_int(k), _ptr(workspace), C.c_size_t(workspace.numel()),
                                    _stream()))
    return out


class DitModel:
    """b2_dit_model over torch tensors: `blocks` a list of BlockWeights, the rest device tensors (kept alive here)."""

    def __init__(self, blocks, F, block_mod_w, block_mod_bias, head_mod_w, head_mod_bias, video_w, video_bias, final_norm,
                 final_w, final_bias, D=3072, heads=24, ext_w=None, ext_bias=None):
        self.keep = (blocks, block_mod_w, block_mod_bias, head_mod_w, head_mod_bias, video_w, video_bias, final_norm, final_w,
                     final_bias, ext_w, ext_bias)
        self.arr = (_lib.BlockWeights * max(1, len(blocks)))(*[b.struct for b in blocks])
        m = _lib.DitModel()
        m.struct_size, m.blocks, m.num_blocks = C.sizeof(_lib.DitModel), self.arr, len(blocks)
        m.D, m.F, m.heads, m.latent_channels = D, F, heads, 128
        p = lambda t: None if t is None else t.data_ptr()
        m.block_mod_w, m.block_mod_bias, m.head_mod_w, m.head_mod_bias = p(block_mod_w), p(block_mod_bias), p(head_mod_w), p(head_mod_bias)
        m.video_w, m.video_bias, m.final_norm, m.final_w, m.final_bias = p(video_w), p(video_bias), p(final_norm), p(final_w), p(final_bias)
        m.ext_w, m.ext_bias, m.ext_channels = p(ext_w), p(ext_bias), 0 if ext_w is None else ext_w.shape[1] - 128
        self.struct = m


def silu_bf16(x, out=None):
    """kernels::silu: bf16(x / (1 + expf(-x)))."""
    out = torch.empty_like(x) if out is None else out
    check(_lib.lib().b2_silu_bf16(_ptr(x), _ptr(out), x.numel(), _stream()))
    return out


def time_modulation_bf16(in_w, in_bias, out_w, out_bias, block_mod_w, block_mod_bias, head_mod_w, head_mod_bias, timestep):
    """MossDit::time_modulation in its bf16 form: (mod bf16 [6 D], head bf16 [2 D]) on the device. All arguments bf16 device tensors
    (a bias may be None)."""
    m = _lib.TimeMlpBf16()
    m.struct_size, m.dim = C.sizeof(_lib.TimeMlpBf16), out_w.shape[0]
    for name, t in (("in_w", in_w), ("in_bias", in_bias), ("out_w", out_w), ("out_bias", out_bias), ("block_mod_w", block_mod_w),
                    ("block_mod_bias", block_mod_bias), ("head_mod_w", head_mod_w), ("head_mod_bias", head_mod_bias)):
        setattr(m, name, None if t is None else t.data_ptr())
    D = out_w.shape[0]
    mod = torch.empty(6 * D, dtype=torch.bfloat16, device=out_w.device)
    head = torch.empty(2 * D, dtype=torch.bfloat16, device=out_w.device)
    ws = torch.empty(_lib.lib().b2_time_modulation_bf16_workspace_bytes(C.byref(m)), dtype=torch.uint8, device=out_w.device)
    check(_lib.lib().b2_time_modulation_bf16(C.byref(m), C.c_float(timestep), _ptr(mod), _ptr(head), _ptr(ws), ws.numel(), _stream()))
    return mod, head


class DitGraphs:
    """b2_dit_graphs: CUDA graphs of whole forwards, least recently used first out. Creating one touches no device."""

    def __init__(self, capacity=8):
        self.handle = C.c_void_p()
        check(_lib.lib().b2_dit_graphs_create(capacity, C.byref(self.handle)))
        self.last_replayed = False

    def stats(self):
        st = _lib.DitGraphStats()
        check(_lib.lib().b2_dit_graphs_stats(self.handle, C.byref(st)))
        return {name: int(getattr(st, name)) for name, _ in st._fields_}

    def clear(self):
        check(_lib.lib().b2_dit_graphs_clear(self.handle))

    def close(self):
        if self.handle:
            _lib.lib().b2_dit_graphs_destroy(self.handle)
            self.handle = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def dit_forward(model: DitModel, latents, time_vector, rows, tier=TIER_INT8, workspace=None, extra=None, ref_kv=None,
                graphs=None, outs=None, mod=None, head=None):
    """rows: list of (text bf16 [S, D], skip mask int, latent index). latents f32 [n, 128, h, w]; time_vector numpy f32 [D].
    Returns the per-row outputs f32 [128, h, w] (and the workspace, for reuse). With `graphs` (a DitGraphs) the forward
    goes through b2_dit_forward_graphed on the current (non-default) stream; pass the same `outs` and `workspace` again for
    the call to find its graph."""
    import numpy as np
    n, _, h, w = latents.shape
    if outs is None:
        outs = [torch.empty((128, h, w), dtype=torch.float32, device=latents.device) for _ in rows]
    arr = (_lib.ForwardRow * len(rows))()
    for i, (text, skip, latent) in enumerate(rows):
        arr[i].text, arr[i].text_len, arr[i].skip, arr[i].latent, arr[i].out = text.data_ptr(), text.shape[0], skip, latent, outs[i].data_ptr()
    tv = None if time_vector is None else np.ascontiguousarray(time_vector, np.float32)
    f = _lib.Forward()
    f.struct_size, f.latents, f.num_latents, f.height, f.width = C.sizeof(_lib.Forward), latents.data_ptr(), n, h, w
    f.time_vector, f.rows, f.num_rows, f.tier = (None if tv is None else tv.ctypes.data), arr, len(rows), tier
    f.mod, f.head = (None if mod is None else mod.data_ptr()), (None if head is None else head.data_ptr())
    f.attention = _lib.AttentionOptions(ATTENTION_Q8_FP8_F32ACC, 0.0, 0.0)
    f.extra = None if extra is None else extra.data_ptr()
    f.ref_kv, f.ref_tokens = (None, 0) if ref_kv is None else (ref_kv.data_ptr(), ref_kv.shape[1])
    need = _lib.lib().b2_dit_forward_workspace_bytes(C.byref(model.struct), C.byref(f))
    if need == 0:
        check(-1)
    if workspace is None or workspace.numel() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=latents.device)
    f.workspace, f.workspace_bytes = workspace.data_ptr(), workspace.numel()
    if graphs is None:
        check(_lib.lib().b2_dit_forward(C.byref(model.struct), C.byref(f), _stream()))
    else:
        replayed = C.c_int(0)
        check(_lib.lib().b2_dit_forward_graphed(graphs.handle, C.byref(model.struct), C.byref(f), _stream(), C.byref(replayed)))
        graphs.last_replayed = bool(replayed.value)
    return outs, workspace


def dit_prefill_references(model, latents, time_vector, tier=TIER_INT8):
    """latents: list of f32 [128, h, w] reference latents. Returns the cache bf16 [num_blocks, sum h w, 2 D]."""
    import numpy as np
    n = len(latents)
    ptrs = (C.c_void_p * n)(*[t.data_ptr() for t in latents])
    hs, ws = (C.c_int * n)(*[t.shape[1] for t in latents]), (C.c_int * n)(*[t.shape[2] for t in latents])
    total = sum(t.shape[1] * t.shape[2] for t in latents)
    m = model.struct
    kv = torch.empty((m.num_blocks, total, 2 * m.D), dtype=torch.bfloat16, device=latents[0].device)
    tv = np.ascontiguousarray(time_vector, np.float32)
    f = _lib.Prefill()
    f.struct_size, f.latents, f.heights, f.widths, f.num_refs = C.sizeof(_lib.Prefill), ptrs, hs, ws, n
    f.time_vector, f.kv_out, f.tier = tv.ctypes.data, kv.data_ptr(), tier
    f.attention = _lib.AttentionOptions(ATTENTION_Q8_FP8_F32ACC, 0.0, 0.0)
    need = _lib.lib().b2_dit_prefill_workspace_bytes(C.byref(m), C.byref(f))
    if need == 0:
        check(-1)
    ws_buf = torch.empty(need, dtype=torch.uint8, device=latents[0].device)
    f.workspace, f.workspace_bytes = ws_buf.data_ptr(), need
    check(_lib.lib().b2_dit_prefill_references(C.byref(m), C.byref(f), _stream()))
    return kv


# ------------------------------------------------------------------------------------------------ paged key-value cache

_DTYPES = {torch.bfloat16: 0, torch.float16: 1}
_PAGED_BYTES = C.sizeof(_lib.PagedCache)

# (A single token's kernels take a few microseconds, so what a call does on the host is a good part of it: the checks below
# are written for their number of tensor queries, and the structs filled in one go.)


try:  # (private names, which another torch may not have)
    _get_device, _get_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
except AttributeError:
    _get_device = _get_stream = None


def _raw_stream() -> int:
    """The current stream's handle as an int; for calls on tensors that are on the GPU already."""
    return torch.cuda.current_stream().cuda_stream if _get_stream is None else _get_stream(_get_device())


@functools.lru_cache(maxsize=1024)
def _workspace_need(call, *shape):
    """Bytes of workspace by the C function `call`, which looks at sizes only: the struct has addresses that nothing follows."""
    batch, kv_heads, page_size, head_dim, slots, dtype = shape[:6]
    dims = page_size * head_dim
    cache = _lib.PagedCache(_PAGED_BYTES, 256, 256, kv_heads * dims, dims, head_dim, 1, _DTYPES[dtype], kv_heads, page_size, head_dim, 256, slots // page_size,
                            slots // page_size, 256, batch)
    n = getattr(_lib.lib(), call)(cache, *shape[6:])
    if n == 0:
        check(-1)
    return n


def _at(t) -> int:
    return 0 if t is None else t.data_ptr()


def _rows(t, name, dtype):
    """(rows, row stride) of a matrix of `dtype` whose rows are contiguous."""
    if t.dtype != dtype or t.dim() != 2:
        raise ValueError(f"{name} must be a {dtype} matrix")
    rows, width = t.shape
    if t.is_contiguous():
        return rows, width
    stride, inner = t.stride()
    if inner != 1 and width > 1:
        raise ValueError(f"the rows of {name} must be contiguous")
    if stride < width and rows > 1:
        raise ValueError(f"the rows of {name} must not overlap")
    return rows, max(stride, width)


def _vector(t, name, count):
    if t.dtype != torch.int32 or t.dim() != 1 or t.numel() != count or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of {count} entries")
    return t.data_ptr()


class PagedCache:
    """b2_paged_cache: pools k and v [pages, kv_heads, page_size, head_dim] (bf16 or fp16 views of the same strides, head_dim
    contiguous), block_table int32 [batch, width] and seq_lens int32 [batch] on the device. The struct holds addresses, so the
    contents may change between calls (lengths that grow, pages that are added) without a new handle."""

    def __init__(self, k, v, block_table, seq_lens):
        shape, strides = k.shape, k.stride()
        dtype = k.dtype
        code = _DTYPES.get(dtype)
        if code is None or dtype != v.dtype or len(shape) != 4 or shape != v.shape or strides != v.stride() or strides[3] != 1:
            raise ValueError("k and v must be bf16 or fp16 pools [pages, kv_heads, page_size, head_dim] of the same strides, head_dim contiguous")
        batch, ld = _rows(block_table, "block_table", torch.int32)
        self.k, self.v, self.block_table, self.seq_lens, self.dtype = k, v, block_table, seq_lens, dtype
        pages, self.kv_heads, self.page_size, self.head_dim = shape
        width = block_table.numel() // batch if batch else 0
        self.batch, self.slots = batch, width * self.page_size
        self._sizes = (batch, self.kv_heads, self.page_size, self.head_dim, self.slots, dtype)
        self.struct = _lib.PagedCache(_PAGED_BYTES, k.data_ptr(), v.data_ptr(), strides[0], strides[1], strides[2], pages, code, self.kv_heads,
                                      self.page_size, self.head_dim, block_table.data_ptr(), ld, width, _vector(seq_lens, "seq_lens", batch), batch)


def _heads_view(t, cache, name):
    if t.dim() != 3 or t.dtype != cache.dtype:
        raise ValueError(f"{name} must be a [tokens, heads, head_dim] view of the cache's dtype")
    tokens, heads, dim = t.shape
    row, head, inner = t.stride()
    if dim != cache.head_dim or inner != 1:
        raise ValueError(f"{name} must have the cache's head_dim, contiguous")
    return _lib.View3(t.data_ptr(), tokens, heads, row, head)


def qk_norm_rope_append(qkv, cache, cu_seqlens, q_norm, k_norm, rope, positions=None, eps=1e-6, interleaved=False, out=None):
    """qkv [tokens, (q_heads + 2 kv_heads) * head_dim]: per-head RMS norm of queries and keys (None: none), rotation by the fp32 table
    rope [positions, rot_dim] (sin | cos; None: none), keys and values into the cache's last slots. Returns the queries
    [tokens, q_heads, head_dim] (into `out` when given; qkv's own query part will do)."""
    tokens, ld = _rows(qkv, "qkv", cache.dtype)
    dim = cache.head_dim
    heads, rest = divmod(qkv.shape[1], dim)
    q_heads = heads - 2 * cache.kv_heads
    if rest or q_heads <= 0:
        raise ValueError("qkv must have q_heads + 2 kv_heads heads")
    for norm in (q_norm, k_norm):
        if norm is not None and (norm.dtype != cache.dtype or norm.dim() != 1 or norm.numel() != dim or not norm.is_contiguous()):
            raise ValueError("q_norm and k_norm must be contiguous [head_dim] tensors of the cache's dtype")
    rows = rot = 0
    if rope is not None:
        if rope.dtype != torch.float32 or rope.dim() != 2 or not rope.is_contiguous():
            raise ValueError("rope must be a contiguous fp32 table [positions, rot_dim]")
        rows, rot = rope.shape
    out = torch.empty((tokens, q_heads, dim), dtype=cache.dtype, device=qkv.device) if out is None else out
    view = _heads_view(out, cache, "out")
    if view.tokens != tokens or view.heads != q_heads:
        raise ValueError("out must be a [tokens, q_heads, head_dim] view")
    check(_lib.lib().b2_qk_norm_rope_append(cache.struct, qkv.data_ptr(), ld, tokens, q_heads, _vector(cu_seqlens, "cu_seqlens", cache.batch + 1),
                                            0 if positions is None else _vector(positions, "positions", tokens), _at(q_norm), _at(k_norm), eps,
                                            _at(rope), rows, rot, interleaved, view.data, view.row_stride, view.head_stride, _raw_stream()))
    return out


def _out_of(q, out, view, cache):
    """The output for q, and its view. (empty_like and empty_strided take half the time of new_empty: a microsecond each.)"""
    if out is not None:
        return out, _heads_view(out, cache, "out")
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    heads, dim = view.heads, cache.head_dim
    return out, _lib.View3(out.data_ptr(), view.tokens, heads, heads * dim, dim)


def _lse_of(q, lse):
    if lse is None:
        tokens, heads, _ = q.shape
        return torch.empty_strided((tokens, heads), (heads, 1), dtype=torch.float32, device=q.device)
    if lse.dtype != torch.float32 or lse.shape != q.shape[:2] or not lse.is_contiguous():
        raise ValueError("lse must be a contiguous fp32 [tokens, q_heads] tensor")
    return lse


def attention_paged_workspace_bytes(cache, tokens, q_heads, max_q, window=0, sinks=0) -> int:
    return _workspace_need("b2_attention_paged_workspace_bytes", *cache._sizes, tokens, q_heads, max_q, window, sinks)


def attention_paged(q, cache, cu_seqlens, max_q, scale, window=0, sinks=0, out=None, lse=None, workspace=None):
    """Causal attention of a prompt's tokens q [tokens, q_heads, head_dim] over the cache that holds their keys and values already;
    with a window the last `window` slots and the first `sinks`. Returns (out, lse): lse fp32 [tokens, q_heads]."""
    view = _heads_view(q, cache, "q")
    out, out_view = _out_of(q, out, view, cache)
    lse = _lse_of(q, lse)
    if workspace is None:
        need = attention_paged_workspace_bytes(cache, view.tokens, view.heads, max_q, window, sinks)
        workspace = q.new_empty(need, dtype=torch.uint8) if need > 256 else None  # (256: none is used)
    check(_lib.lib().b2_attention_paged(cache.struct, view, out_view, lse.data_ptr(), _vector(cu_seqlens, "cu_seqlens", cache.batch + 1),
                                        max_q, scale, window, sinks, _at(workspace), 0 if workspace is None else workspace.numel(), _raw_stream()))
    return out, lse


def attention_paged_decode_workspace_bytes(cache, q_heads, max_len=0, window=0, sinks=0, weights=False) -> int:
    return _workspace_need("b2_attention_paged_decode_workspace_bytes", *cache._sizes, q_heads, max_len, window, sinks, weights)


def attention_paged_decode(q, cache, scale, max_len=0, window=0, sinks=0, weights=None, weights_out=None, out=None, lse=None, workspace=None):
    """Attention of one new token per sequence, q [batch, q_heads, head_dim], split over the cache's length. With `weights` (fp32 [batch,
    kv_heads, slots]) the attention each slot got is added to them (in weights_out, or in place). Returns (out, lse)."""
    view = _heads_view(q, cache, "q")
    out, out_view = _out_of(q, out, view, cache)
    lse = _lse_of(q, lse)
    ld = 0
    if weights is not None:
        weights_out = weights if weights_out is None else weights_out
        ld = _slots_of(weights, cache, "weights")
        if weights_out is not weights and _slots_of(weights_out, cache, "weights_out") != ld:
            raise ValueError("weights and weights_out must have the same shape")
    if workspace is None:
        need = attention_paged_decode_workspace_bytes(cache, view.heads, max_len, window, sinks, weights is not None)
        workspace = q.new_empty(need, dtype=torch.uint8) if need > 256 else None  # (256: none is used)
    check(_lib.lib().b2_attention_paged_decode(cache.struct, view, out_view, lse.data_ptr(), max_len, scale, window, sinks,
                                               _at(weights), _at(weights_out), ld, _at(workspace), 0 if workspace is None else workspace.numel(), _raw_stream()))
    return out, lse


def _slots_of(t, cache, name):
    """Slots of a contiguous fp32 [batch, kv_heads, slots] tensor."""
    if t.dtype != torch.float32 or t.dim() != 3 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous fp32 [batch, kv_heads, slots] tensor")
    batch, heads, slots = t.shape
    if batch != cache.batch or heads != cache.kv_heads:
        raise ValueError(f"{name} must have a row for each sequence and key head")
    return slots


def kv_evict(cache, weights, table_out, budget, sinks=0, recent=0, kept=None, lens_out=None, weights_out=None):
    """Sequences of more than `budget` slots keep their first `sinks`, their last `recent` and, of the rest, the slots of most weight
    (fp32 [batch, kv_heads, slots]), for each key head by itself; what is kept moves in order to the pages of table_out. Returns
    (kept int32 [batch, kv_heads, budget], lens int32 [batch], not the cache's own); weights_out receives the weights of what is kept."""
    if budget <= 0:
        raise ValueError("budget must be positive")
    slots = _slots_of(weights, cache, "weights")
    rows_out, ld_out = _rows(table_out, "table_out", torch.int32)
    if rows_out != cache.batch:
        raise ValueError("table_out must have a row for every sequence")
    slots_out = 0 if weights_out is None else _slots_of(weights_out, cache, "weights_out")
    if kept is None:
        kept = torch.empty_strided((cache.batch, cache.kv_heads, budget), (cache.kv_heads * budget, budget, 1), dtype=torch.int32, device=weights.device)
    lens_out = torch.empty_like(cache.seq_lens) if lens_out is None else lens_out
    if kept.dtype != torch.int32 or kept.shape != (cache.batch, cache.kv_heads, budget) or not kept.is_contiguous():
        raise ValueError("kept must be a contiguous int32 [batch, kv_heads, budget] tensor")
    check(_lib.lib().b2_kv_evict(cache.struct, weights.data_ptr(), slots, sinks, recent, budget, table_out.data_ptr(), ld_out, table_out.shape[1],
                                 kept.data_ptr(), _vector(lens_out, "lens_out", cache.batch), _at(weights_out), slots_out, _raw_stream()))
    return kept, lens_out


def paged_cache_status(clear=False) -> int:
    """Bits that the kernels on paged caches raised (b2_paged_cache_status): 0 when every length, page and position was in bounds."""
    v = C.c_uint(0)
    check(_lib.lib().b2_paged_cache_status(C.byref(v), int(clear)))
    return int(v.value)


# ------------------------------------------------------------------------------------------------ around a text decoder's attention

_DTYPES_ALL = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_CODES = {torch.int8: 0, torch.float8_e4m3fn: 1}
_NORM_BYTES, _LOGPROBS_BYTES, _LORA_BYTES = C.sizeof(_lib.NormQuantize), C.sizeof(_lib.Logprobs), C.sizeof(_lib.Lora)


def _here(first, *others):
    """All tensors that are given lie on the current CUDA device."""
    at = first.get_device()
    if at < 0 or at != (torch.cuda.current_device() if _get_device is None else _get_device()):
        raise ValueError("the tensors must be on the current CUDA device")
    for t in others:
        if t is not None and t.get_device() != at:
            raise ValueError("the tensors must be on the current CUDA device")


def _like(t, name, shape, dtypes):
    """Row stride of a matrix of this shape, of one of `dtypes`, whose rows are contiguous."""
    if t.dtype not in dtypes or t.shape != shape:
        raise ValueError(f"{name} must be a {list(shape)} matrix of {' or '.join(map(str, dtypes))}")
    return shape[1] if t.is_contiguous() else _rows(t, name, t.dtype)[1]


def add_rms_norm_quantize(x, weight=None, residual=None, eps=1e-6, dtype=torch.int8, group=0, residual_out=None, norm_out=None, q=None, scale=None):
    """The sum s = x + residual ([tokens, dim]; into residual_out, or the residual itself) and its root-mean-square norm times weight [dim] in 8 bits
    for the projection that follows: codes of `dtype` (int8 or float8_e4m3fn) with an fp32 scale per token, or per `group` channels
    (32, 64, 128 or 256). x bf16, fp16 or fp32, the residual of x's type or fp32. norm_out (bf16 or fp16 [tokens, dim]) receives the norm
    unquantised besides, for adapters. Returns (q, scale): scale [tokens], or [tokens, dim / group]."""
    types = _DTYPES_ALL
    x_dtype = x.dtype
    code, codes = types.get(x_dtype), _CODES.get(dtype)
    if code is None or codes is None:
        raise ValueError("x must be bf16, fp16 or fp32, the codes int8 or float8_e4m3fn")
    tokens, ldx = _rows(x, "x", x_dtype)
    shape, device = x.shape, x.device
    dim = shape[1]
    if group < 0 or (group and dim % group):
        raise ValueError("group must be 0, 32, 64, 128 or 256 and divide dim")
    ld_res = ld_res_out = ld_norm = at_res = at_res_out = r_code = 0
    if residual is not None:
        ld_res = ld_res_out = _like(residual, "residual", shape, (x_dtype, torch.float32))
        r_code, at_res = types[residual.dtype], residual.data_ptr()
        if residual_out is None:
            at_res_out = at_res
        else:
            ld_res_out, at_res_out = _like(residual_out, "residual_out", shape, (residual.dtype,)), residual_out.data_ptr()
    elif residual_out is not None:
        raise ValueError("residual_out needs a residual")
    if norm_out is not None:
        ld_norm = _like(norm_out, "norm_out", shape, (torch.bfloat16, torch.float16))
    if weight is not None and (weight.dtype not in types or weight.dim() != 1 or weight.numel() != dim or not weight.is_contiguous()):
        raise ValueError("weight must be a contiguous [dim] tensor of bf16, fp16 or fp32")
    ldq = dim if q is None else _like(q, "q", shape, (dtype,))
    if scale is not None and (scale.dtype != torch.float32 or scale.shape != ((tokens, dim // group) if group else (tokens,)) or not scale.is_contiguous()):
        raise ValueError("scale must be a contiguous fp32 tensor [tokens], or [tokens, dim / group]")
    _here(x, residual, residual_out, norm_out, weight, q, scale)
    # (empty_strided takes half of empty's time, a microsecond.)
    if q is None:
        q = torch.empty_strided(shape, (dim, 1), dtype=dtype, device=device)
    if scale is None:
        groups = dim // group if group else 1
        scale = torch.empty_strided((tokens, groups) if group else (tokens,), (groups, 1) if group else (1,), dtype=torch.float32, device=device)
    check(_lib.lib().b2_add_rms_norm_quantize(
        _lib.NormQuantize(_NORM_BYTES, tokens, dim, group, eps, codes, x.data_ptr(), ldx, at_res, ld_res, at_res_out, ld_res_out,
                          0 if weight is None else weight.data_ptr(), 0 if norm_out is None else norm_out.data_ptr(), ld_norm, q.data_ptr(), ldq, scale.data_ptr(),
                          code, r_code, 0 if weight is None else types[weight.dtype], 0 if norm_out is None else types[norm_out.dtype]), _raw_stream()))
    return q, scale


class TokenLogprobs(typing.NamedTuple):
    """What token_logprobs returns; logprobs and ranks are None without targets, the last two without alternatives."""
    logprobs: typing.Optional[torch.Tensor]      # fp32 [rows]
    ranks: typing.Optional[torch.Tensor]         # int32 [rows], from 1
    entropy: torch.Tensor                        # fp32 [rows]
    lse: torch.Tensor                            # fp32 [rows]
    top_logprobs: typing.Optional[torch.Tensor]  # fp32 [rows, top]
    top_tokens: typing.Optional[torch.Tensor]    # int32 [rows, top]


def token_logprobs(logits, targets=None, top=0, scale=1.0):
    """Of logits [rows, vocab] (bf16, fp16 or fp32 rows of any stride) times scale (one over the temperature): the log probability and the rank
    of targets (int64 [rows]; a negative one is none and has 0 for both), the entropy, the log of the sum of exponentials, and the `top` (up to 32)
    most probable tokens with their log probabilities, equal ones by number. Returns TokenLogprobs."""
    code = _DTYPES_ALL.get(logits.dtype)
    if code is None:
        raise ValueError("logits must be bf16, fp16 or fp32")
    rows, ld = _rows(logits, "logits", logits.dtype)
    if targets is not None and (targets.dtype != torch.int64 or targets.dim() != 1 or targets.numel() != rows or not targets.is_contiguous()):
        raise ValueError("targets must be a contiguous int64 [rows] tensor")
    if top < 0 or top > 32:
        raise ValueError("top must be from 0 to 32 and at most vocab")
    _here(logits, targets)
    device, new, one = logits.device, torch.empty_strided, (1,)
    entropy = new((rows,), one, dtype=torch.float32, device=device)
    lse = torch.empty_like(entropy)
    logprobs = ranks = top_logprobs = top_tokens = None
    at = [0, 0, 0, 0]
    if targets is not None:
        logprobs, ranks = torch.empty_like(entropy), new((rows,), one, dtype=torch.int32, device=device)
        at[0], at[1] = logprobs.data_ptr(), ranks.data_ptr()
    if top:
        top_logprobs = new((rows, top), (top, 1), dtype=torch.float32, device=device)
        top_tokens = new((rows, top), (top, 1), dtype=torch.int32, device=device)
        at[2], at[3] = top_logprobs.data_ptr(), top_tokens.data_ptr()
    check(_lib.lib().b2_token_logprobs(
        _lib.Logprobs(_LOGPROBS_BYTES, logits.data_ptr(), ld, rows, code, logits.shape[1], top, scale, 0 if targets is None else targets.data_ptr(), at[0], at[1],
                      entropy.data_ptr(), lse.data_ptr(), at[2], at[3]), _raw_stream()))
    return TokenLogprobs(logprobs, ranks, entropy, lse, top_logprobs, top_tokens)


class LoraAdapters:
    """b2_lora: the low-rank adapters of one projection, a [adapters, rank, dim] and b [adapters, width, rank] (bf16 or fp16, rows contiguous), scales
    fp32 [adapters] (None: 1) and, where some have a lower rank than the tensors, ranks int32 [adapters]. The struct holds addresses, so the
    contents may change between calls."""

    def __init__(self, a, b, scales=None, ranks=None):
        code = _DTYPES.get(a.dtype)
        if code is None or a.dtype != b.dtype or a.dim() != 3 or b.dim() != 3 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2]:
            raise ValueError("a and b must be bf16 or fp16 tensors [adapters, rank, dim] and [adapters, width, rank]")
        n, rank, dim = a.shape
        for name, t in (("a", a), ("b", b)):
            if (t.stride(2) != 1 and t.shape[2] > 1) or (t.stride(1) < t.shape[2] and t.shape[1] > 1):
                raise ValueError(f"the rows of {name} must be contiguous and not overlap")
        if scales is not None and (scales.dtype != torch.float32 or scales.dim() != 1 or scales.numel() != n or not scales.is_contiguous()):
            raise ValueError("scales must be a contiguous fp32 [adapters] tensor")
        if ranks is not None:
            _vector(ranks, "ranks", n)
        for name, t in (("b", b), ("scales", scales), ("ranks", ranks)):
            if t is not None and t.device != a.device:
                raise ValueError(f"{name} must be on a's device")
        self.a, self.b, self.scales, self.ranks, self.dtype, self.dtypes, self.device = a, b, scales, ranks, a.dtype, (a.dtype,), a.device
        self.adapters, self.rank, self.dim, self.width = n, rank, dim, b.shape[1]
        self.struct = _lib.Lora(_LORA_BYTES, a.data_ptr(), b.data_ptr(), a.stride(0), max(a.stride(1), dim), b.stride(0), max(b.stride(1), rank), _at(scales),
                                _at(ranks), dim, self.width, n, rank, code)


class LoraPlan:
    """b2_lora_plan: a step's tokens sorted by their adapter, token_adapters int32 [tokens] (negative: none), for every lora_add of the step. Where
    the tensor's contents change, fill() sorts them anew (on the current stream; it can be captured along with the calls that use it)."""

    def __init__(self, token_adapters, adapters):
        self.tokens, self.adapters, self.token_adapters = token_adapters.numel(), adapters, token_adapters
        _vector(token_adapters, "token_adapters", self.tokens)
        self._sizes = {}
        need = _lib.lib().b2_lora_plan_bytes(self.tokens, adapters)
        if need == 0:
            check(-1)
        _here(token_adapters)
        self.device, self.bytes = token_adapters.device, need
        self.buffer = torch.empty(need, dtype=torch.uint8, device=self.device)
        self.at = self.buffer.data_ptr()
        self.fill()

    def fill(self):
        _here(self.buffer, self.token_adapters)
        check(_lib.lib().b2_lora_plan(self.token_adapters.data_ptr(), self.tokens, self.adapters, self.at, self.bytes, _raw_stream()))

    def workspace_bytes(self, dim, rank) -> int:
        need = self._sizes.get((dim, rank))
        if need is None:
            need = _lib.lib().b2_lora_workspace_bytes(self.tokens, self.adapters, dim, rank)
            if need == 0:
                check(-1)
            self._sizes[(dim, rank)] = need
        return need


def lora_add(y, x, adapters, plan, out=None, workspace=None):
    """y [tokens, width] plus, for each token with an adapter, scale (x A^T) B^T of its row of x [tokens, dim]: in y's place, or into `out`. y and x
    are views with contiguous rows (a slice of a fused projection's columns, say). Returns out."""
    tokens, dtypes = plan.tokens, adapters.dtypes
    if plan.adapters != adapters.adapters:
        raise ValueError("the plan is of another number of adapters")
    ldx = _like(x, "x", (tokens, adapters.dim), dtypes)
    ldy = ldo = _like(y, "y", (tokens, adapters.width), dtypes)
    if out is None:
        out = y
    else:
        ldo = _like(out, "out", (tokens, adapters.width), dtypes)
    if workspace is not None and not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")
    _here(y, x, out, adapters.a, plan.buffer, workspace)
    need = plan.workspace_bytes(adapters.dim, adapters.rank)
    if workspace is not None:
        given = workspace.numel() * workspace.element_size()
    elif need > 256:
        workspace, given = torch.empty_strided((need,), (1,), dtype=torch.uint8, device=plan.device), need
    else:
        given = 0  # (256: none is used)
    check(_lib.lib().b2_lora_add(adapters.struct, plan.at, plan.bytes, tokens, x.data_ptr(), ldx, y.data_ptr(), ldy, out.data_ptr(), ldo, _at(workspace), given,
                                 _raw_stream()))
    return out


def lora_status(clear=False) -> int:
    """Bits that the kernels on adapters raised (b2_lora_status): 0 when every adapter, rank and plan was as it should be."""
    v = C.c_uint(0)
    check(_lib.lib().b2_lora_status(C.byref(v), int(clear)))
    return int(v.value)


# ------------------------------------------------------------------------------------------------ weight ingestion

class _Loaded:
    """A struct that lives in a loaded file (b2_block_weights or b2_dit_model): `.struct` for the calls that take one."""

    def __init__(self, struct, owner):
        self.struct, self.owner = struct, owner


class DitFile:
    """b2_dit_file: the quantized DiT of a ComfyUI-layout safetensors file, on the current device."""

    def __init__(self, path: str, expanded: bool = False):
        """expanded: grouped 4-bit (W4A8) weights are expanded to the INT8 grid once at load (b2_dit_file_open_expanded)."""
        self.handle = C.c_void_p()
        opener = _lib.lib().b2_dit_file_open_expanded if expanded else _lib.lib().b2_dit_file_open
        check(opener(str(path).encode(), C.byref(self.handle)))
        info = _lib.DitFileInfo()
        info.struct_size = C.sizeof(_lib.DitFileInfo)
        check(_lib.lib().b2_dit_file_get_info(self.handle, C.byref(info)))
        self.num_blocks, self.F, self.tier, self.stored_tier = info.num_blocks, info.F, info.tier, info.stored_tier
        self.has_shell, self.has_time_embedding, self.device_bytes = bool(info.has_shell), bool(info.has_time_embedding), info.device_bytes
        model = _lib.lib().b2_dit_file_model(self.handle).contents
        self.model = _Loaded(model, self)
        self.blocks = [_Loaded(model.blocks[i], self) for i in range(self.num_blocks)]

    def time_vector(self, timestep: float):
        import numpy as np
        te = _lib.lib().b2_dit_file_time_embedding(self.handle)
        if not te:
            raise ValueError("the file has no time embedding")
        out = np.empty(te.contents.dim, np.float32)
        check(_lib.lib().b2_time_vector_fp32(te, C.c_float(timestep), out.ctypes.data_as(C.c_void_p)))
        return out

    def time_modulation_bf16(self, timestep: float):
        """(mod bf16 [6 D], head bf16 [2 D]) through the bf16 form of the file's timestep MLP and modulation linears."""
        m = _lib.lib().b2_dit_file_time_mlp_bf16(self.handle)
        if not m:
            raise ValueError("the file lacks the shell or the time embedding")
        D = m.contents.dim
        mod = torch.empty(6 * D, dtype=torch.bfloat16, device="cuda")
        head = torch.empty(2 * D, dtype=torch.bfloat16, device="cuda")
        ws = torch.empty(_lib.lib().b2_time_modulation_bf16_workspace_bytes(m), dtype=torch.uint8, device="cuda")
        check(_lib.lib().b2_time_modulation_bf16(m, C.c_float(timestep), _ptr(mod), _ptr(head), _ptr(ws), ws.numel(), _stream()))
        return mod, head

    def close(self):
        if self.handle:
            _lib.lib().b2_dit_file_close(self.handle)
            self.handle = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
