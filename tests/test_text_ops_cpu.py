"""What the operators around a text decoder's attention refuse, before any launch (no GPU is needed: addresses are never followed)."""
import ctypes as C
import math

import pytest
import torch

from owoinfer_b200 import _lib, ops

A = 0x10000  # a 256-byte aligned address that nothing reads
BF16, F16, F32 = 0, 1, 2


def norm(**over):
    v = dict(struct_size=C.sizeof(_lib.NormQuantize), tokens=1, dim=64, group=0, eps=1e-6, codes=0, x=A, ldx=64, residual=A, ld_residual=64, residual_out=A,
             ld_residual_out=64, weight=A, norm_out=A, ld_norm=64, q=A, ldq=64, scale=A, x_dtype=BF16, residual_dtype=F32, weight_dtype=BF16, norm_dtype=BF16)
    v.update(over)
    return _lib.lib().b2_add_rms_norm_quantize(_lib.NormQuantize(*(v[name] for name, _ in _lib.NormQuantize._fields_)), None)


def logprobs(**over):
    v = dict(struct_size=C.sizeof(_lib.Logprobs), logits=A, ld=100, rows=1, dtype=BF16, vocab=100, top=5, scale=1.0, targets=A, logprobs=A, ranks=A, entropy=A,
             lse=A, top_logprobs=A, top_tokens=A)
    v.update(over)
    return _lib.lib().b2_token_logprobs(_lib.Logprobs(*(v[name] for name, _ in _lib.Logprobs._fields_)), None)


def lora(plan=A, plan_bytes=1 << 20, tokens=4, x=A, ldx=64, y=A, ldy=128, out=A + 4096, ldo=128, ws=A, ws_bytes=1 << 20, **over):
    v = dict(struct_size=C.sizeof(_lib.Lora), a=A, b=A, a_adapter_stride=16 * 64, a_row_stride=64, b_adapter_stride=128 * 16, b_row_stride=16, scales=A, ranks=None,
             dim=64, width=128, adapters=3, rank=16, dtype=BF16)
    v.update(over)
    return _lib.lib().b2_lora_add(_lib.Lora(*(v[name] for name, _ in _lib.Lora._fields_)), plan, plan_bytes, tokens, x, ldx, y, ldy, out, ldo, ws, ws_bytes, None)


def plan(ids=A, tokens=4, adapters=3, at=A, size=1 << 20):
    return _lib.lib().b2_lora_plan(ids, tokens, adapters, at, size, None)


@pytest.mark.parametrize("call,over,word", [
    (norm, dict(struct_size=8), "struct_size"), (norm, dict(tokens=-1), "tokens"), (norm, dict(tokens=1 << 31), "tokens"), (norm, dict(dim=60), "dim"),
    (norm, dict(dim=0), "dim"), (norm, dict(dim=32776), "dim"), (norm, dict(group=48), "group"), (norm, dict(group=128), "group"), (norm, dict(group=-32), "group"),
    (norm, dict(eps=-1e-9), "eps"), (norm, dict(eps=math.nan), "eps"), (norm, dict(eps=math.inf), "eps"), (norm, dict(codes=2), "codes"), (norm, dict(x_dtype=3), "x_dtype"),
    (norm, dict(residual=None), "residual_out"), (norm, dict(residual_dtype=F16), "residual"), (norm, dict(weight_dtype=5), "weight_dtype"), (norm, dict(norm_dtype=F32), "norm_out"),
    (norm, dict(x=None), "x must"), (norm, dict(x=A + 8), "x must"), (norm, dict(ldx=60), "x must"), (norm, dict(ldx=68), "x must"), (norm, dict(residual=A + 4), "residual must"),
    (norm, dict(ld_residual=66), "residual must"), (norm, dict(residual_out=A + 4), "residual_out must"), (norm, dict(norm_out=A + 2), "norm_out must"),
    (norm, dict(ld_norm=32), "norm_out must"), (norm, dict(weight=A + 2), "weight"), (norm, dict(q=None), "q must"), (norm, dict(q=A + 4), "q must"), (norm, dict(ldq=68), "q must"),
    (norm, dict(scale=None), "scale"), (norm, dict(scale=A + 2), "scale"),
    (logprobs, dict(struct_size=8), "struct_size"), (logprobs, dict(dtype=3), "dtype"), (logprobs, dict(rows=-1), "rows"), (logprobs, dict(rows=1 << 31), "rows"),
    (logprobs, dict(vocab=0), "vocab"), (logprobs, dict(vocab=(1 << 30) + 1), "vocab"), (logprobs, dict(top=-1), "top"), (logprobs, dict(top=33), "top"),
    (logprobs, dict(top=20, vocab=19), "top"), (logprobs, dict(scale=0.0), "scale"), (logprobs, dict(scale=-1.0), "scale"), (logprobs, dict(scale=math.nan), "scale"),
    (logprobs, dict(scale=math.inf), "scale"), (logprobs, dict(logits=None), "logits"), (logprobs, dict(logits=A + 1), "logits"), (logprobs, dict(ld=99), "logits"),
    (logprobs, dict(logits=A + 2, dtype=F32), "logits"), (logprobs, dict(top_tokens=None), "top_"), (logprobs, dict(top_logprobs=None), "top_"),
    (logprobs, dict(lse=A + 2), "output"), (logprobs, dict(targets=A + 4), "targets"),
    (lora, dict(struct_size=8), "struct_size"), (lora, dict(dtype=F32), "dtype"), (lora, dict(tokens=-1), "tokens"), (lora, dict(adapters=0), "adapters"),
    (lora, dict(adapters=4097), "adapters"), (lora, dict(dim=60), "dim"), (lora, dict(width=12), "width"), (lora, dict(rank=12), "rank"), (lora, dict(rank=136), "rank"),
    (lora, dict(a=None), "a must"), (lora, dict(a_row_stride=56), "a must"), (lora, dict(a_row_stride=68), "a must"), (lora, dict(a_adapter_stride=4), "a must"),
    (lora, dict(b=A + 8), "b must"), (lora, dict(b_row_stride=8), "b must"), (lora, dict(b_adapter_stride=-8), "b must"), (lora, dict(scales=A + 2), "scales"),
    (lora, dict(ranks=A + 2), "ranks"), (lora, dict(plan=None), "plan"), (lora, dict(plan=A + 64), "plan"), (lora, dict(plan_bytes=16), "plan"), (lora, dict(x=A + 2), "x must"),
    (lora, dict(ldx=60), "x must"), (lora, dict(y=None), "y must"), (lora, dict(ldy=120), "y must"), (lora, dict(out=A + 8), "out must"), (lora, dict(ldo=132), "out must"),
    (lora, dict(out=A, ldo=136), "y's"), (lora, dict(out=A, y=A + 4096), "x's"), (lora, dict(ws=None), "workspace"), (lora, dict(ws_bytes=64), "workspace"), (lora, dict(ws=A + 128), "workspace"),
    (lora, dict(tokens=20000, plan_bytes=1 << 22, ws_bytes=4096), "workspace"), (lora, dict(tokens=20000, plan_bytes=1 << 22, ws=None, ws_bytes=0), "workspace"),
    (plan, dict(tokens=-1), "tokens"), (plan, dict(adapters=0), "adapters"), (plan, dict(at=None), "plan"), (plan, dict(size=0), "plan"), (plan, dict(at=A + 16), "plan"),
    (plan, dict(ids=None), "token_adapters"), (plan, dict(ids=A + 2), "token_adapters"),
], ids=lambda v: v.__name__ if callable(v) else "-".join(f"{k}={x}" for k, x in v.items()) if isinstance(v, dict) else "")
def test_refusals(call, over, word):
    assert call(**over) == -1
    assert word in _lib.lib().b2_last_error_message().decode()


def test_nothing_to_do_touches_nothing():
    assert norm(tokens=0, x=None, q=None) == 0 and logprobs(rows=0, logits=None) == 0 and lora(tokens=0, x=None, y=None, out=None, plan=None) == 0
    assert plan(tokens=0, ids=None) == 0


@pytest.mark.parametrize("call,args", [("b2_lora_plan_bytes", (-1, 1)), ("b2_lora_plan_bytes", (1, 0)), ("b2_lora_workspace_bytes", (1, 1, 12, 8)), ("b2_lora_workspace_bytes", (1, 1, 16, 4))])
def test_sizes_of_invalid_arguments(call, args):
    assert getattr(_lib.lib(), call)(*args) == 0


def test_sizes():
    lib = _lib.lib()
    for tokens in (0, 1, 16, 17, 1024, 1025, 100000):
        for adapters in (1, 64, 4096):
            assert lib.b2_lora_plan_bytes(tokens, adapters) >= 16 + 4 * tokens
            assert lib.b2_lora_workspace_bytes(tokens, adapters, 4096, 128) >= 256


x = torch.zeros(4, 64, dtype=torch.bfloat16)
ids = torch.zeros(4, dtype=torch.int32)


def adapters(n=3, rank=16, dim=64, width=128, dtype=torch.bfloat16, **how):
    return ops.LoraAdapters(torch.zeros(n, rank, dim, dtype=dtype), torch.zeros(n, width, rank, dtype=dtype), **how)


class Plan:
    tokens, adapters, buffer, device, at, bytes = 4, 3, torch.zeros(512, dtype=torch.uint8), torch.device("cpu"), 0, 512

    def workspace_bytes(self, dim, rank):
        return 256


@pytest.mark.parametrize("call,word", [
    (lambda: ops.add_rms_norm_quantize(x.double()), "x must"), (lambda: ops.add_rms_norm_quantize(x, dtype=torch.uint8), "codes"),
    (lambda: ops.add_rms_norm_quantize(x[0]), "x must"), (lambda: ops.add_rms_norm_quantize(x.t()), "contiguous"), (lambda: ops.add_rms_norm_quantize(x, group=60), "group"),
    (lambda: ops.add_rms_norm_quantize(x, residual=x[:2]), "residual"), (lambda: ops.add_rms_norm_quantize(x, residual=x.half()), "residual"),
    (lambda: ops.add_rms_norm_quantize(x, residual=x[:1].expand(4, 64)), "overlap"), (lambda: ops.add_rms_norm_quantize(x, residual_out=x), "residual_out"),
    (lambda: ops.add_rms_norm_quantize(x, residual=x, residual_out=x.float()), "residual_out"), (lambda: ops.add_rms_norm_quantize(x, norm_out=x.float()), "norm_out"),
    (lambda: ops.add_rms_norm_quantize(x, x), "weight"), (lambda: ops.add_rms_norm_quantize(x, x[0, :32]), "weight"), (lambda: ops.add_rms_norm_quantize(x, q=x), "q must"),
    (lambda: ops.add_rms_norm_quantize(x, scale=torch.zeros(3)), "scale"), (lambda: ops.add_rms_norm_quantize(x), "CUDA"),
    (lambda: ops.token_logprobs(x.long()), "logits"), (lambda: ops.token_logprobs(x[0]), "logits"), (lambda: ops.token_logprobs(x, ids), "targets"),
    (lambda: ops.token_logprobs(x, ids[:3].long()), "targets"), (lambda: ops.token_logprobs(x, top=-1), "top"), (lambda: ops.token_logprobs(x, top=33), "top"),
    (lambda: ops.token_logprobs(x), "CUDA"),
    (lambda: adapters(dtype=torch.float32), "bf16 or fp16"), (lambda: ops.LoraAdapters(torch.zeros(3, 8, 64).half(), torch.zeros(3, 64, 16).half()), "adapters"),
    (lambda: adapters(scales=torch.ones(2)), "scales"), (lambda: adapters(scales=torch.ones(3).double()), "scales"), (lambda: adapters(ranks=torch.ones(3)), "ranks"),
    (lambda: ops.LoraAdapters(torch.zeros(3, 64, 16).half().transpose(1, 2), torch.zeros(3, 64, 16).half()), "contiguous"),
    (lambda: ops.LoraPlan(ids.long(), 3), "token_adapters"), (lambda: ops.LoraPlan(ids, 0), "adapters"), (lambda: ops.LoraPlan(ids, 3), "CUDA"),
    (lambda: ops.lora_add(torch.zeros(4, 128).bfloat16(), x, adapters(2), Plan()), "number of adapters"), (lambda: ops.lora_add(x, x, adapters(), Plan()), "y must"),
    (lambda: ops.lora_add(torch.zeros(4, 128).bfloat16(), x[:3], adapters(), Plan()), "x must"), (lambda: ops.lora_add(torch.zeros(4, 128).half(), x, adapters(), Plan()), "y must"),
    (lambda: ops.lora_add(torch.zeros(4, 128).bfloat16(), x, adapters(), Plan(), out=x), "out must"),
    (lambda: ops.lora_add(torch.zeros(4, 128).bfloat16(), x, adapters(), Plan()), "CUDA"),
])
def test_refusals_of_the_python_calls(call, word):
    with pytest.raises(ValueError, match=word):
        call()
