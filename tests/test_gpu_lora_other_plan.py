"""lora_add with a plan of other tokens or adapters than the call's: nothing is read or written by it, a bit of the status is raised."""
import pytest
import torch

from owoinfer_b200 import ops
from tests.test_gpu_lora import check, exact, make

pytestmark = pytest.mark.gpu


# (each of the ways that a call can go)
@pytest.mark.parametrize("tokens,rank,adapters", [(40, 16, 5), (1500, 32, 4), (17000, 16, 3), (1600, 64, 2)])
@pytest.mark.parametrize("what", ["tokens", "adapters", "not filled"])
def test_a_plan_of_another_size(tokens, rank, adapters, what):
    ops.lora_status(clear=True)
    x, y, a, b, scales, ids = make(tokens, 64, 64, rank, adapters, torch.bfloat16, seed=1)
    plan = ops.LoraPlan(ids, adapters)
    own = ops.LoraAdapters(a, b, scales)
    out = torch.full_like(y, 3.0)
    if what == "tokens":  # (a plan that is large enough, of more tokens than the call has)
        plan.tokens = tokens - 1
        ops.lora_add(y[1:], x[1:], own, plan, out=out[1:])
    elif what == "adapters":
        plan.adapters = adapters - 1
        ops.lora_add(y, x, ops.LoraAdapters(a[1:], b[1:], scales[1:].clone()), plan, out=out)
    else:
        plan.buffer.zero_()
        ops.lora_add(y, x, own, plan, out=out)
    assert (out == 3.0).all() and ops.lora_status(clear=True) == 8
    # ... and filled, it is this call's
    plan.tokens, plan.adapters, plan._sizes = tokens, adapters, {}
    plan.fill()
    want, off = exact(x, y, a, b, scales, ids)
    check(ops.lora_add(y, x, own, plan, out=out), want, off, torch.bfloat16)
    assert ops.lora_status(clear=True) == 0
