"""lora_add against the formula in 64 bits: plans, ranks, views, types, what is not used, what stays as it was."""
import pytest
import torch

from owoinfer_b200 import ops

pytestmark = pytest.mark.gpu
bf16, f16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _status():
    ops.lora_status(clear=True)
    yield
    assert ops.lora_status(clear=True) == 0


def make(tokens, dim, width, rank, adapters, dtype, seed=0, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *shape, s=1.0: (s * torch.randn(shape, generator=g, device="cuda")).to(dtype)  # noqa: E731
    x, y, a, b = n(tokens, dim, s=std), n(tokens, width), n(adapters, rank, dim, s=dim ** -0.5), n(adapters, width, rank, s=rank ** -0.5)
    scales = 0.25 + torch.rand(adapters, generator=g, device="cuda")
    ids = torch.randint(-1, adapters, (tokens,), generator=torch.Generator().manual_seed(seed), dtype=torch.int32).cuda()
    return x, y, a, b, scales, ids


def exact(x, y, a, b, scales, ids, ranks=None):
    """(out, how far it may be off ahead of its own rounding)"""
    out, off = y.double(), torch.zeros(y.shape, dtype=torch.float64, device="cuda")
    # t = x A^T: products are exact in fp32 and added in chains of dim at most, over parts that are joined; its two 16-bit parts hold 16 bits
    # (bf16) of it; t B^T is a chain of rank products of both.
    chain, held = (x.shape[1] + 32) * 2.0 ** -24, 2.0 ** -16
    for n in range(a.shape[0]):
        r = a.shape[1] if ranks is None else int(ranks[n])
        mine = (ids == n).nonzero()[:, 0]
        if len(mine) == 0 or r == 0:
            continue
        xs, an, bn, s = x[mine].double(), a[n, :r].double(), b[n, :, :r].double(), 1.0 if scales is None else float(scales[n])
        t, t_abs = xs @ an.T, xs.abs() @ an.abs().T
        out[mine] += s * (t @ bn.T)
        off[mine] += s * ((chain * t_abs + (held + (2 * r + 8) * 2.0 ** -24) * t.abs()) @ bn.abs().T)
    return out, off


def check(got, want, off, dtype):
    half = torch.finfo(dtype).eps / 2
    assert ((got.double() - want).abs() <= want.abs() * (half + 2.0 ** -23) + 2 * off + 2.0 ** -25).all(), ((got.double() - want).abs() - want.abs() * half - 2 * off).max()


@pytest.mark.parametrize("dtype", [bf16, f16], ids=["bf16", "f16"])
@pytest.mark.parametrize("tokens,dim,width,rank,adapters", [
    (1, 8, 8, 8, 1), (1, 2048, 2048, 16, 4), (15, 64, 24, 16, 3), (16, 40, 136, 24, 1), (17, 520, 1000, 40, 5), (100, 256, 512, 128, 60), (64, 4096, 640, 16, 48),
    (4000, 1032, 200, 128, 6), (2500, 264, 72, 64, 50), (3000, 520, 1000, 24, 200), (500, 520, 264, 8, 450), (6000, 512, 72, 32, 90), (900, 1544, 520, 128, 30),
    (64, 136, 264, 128, 40), (1024, 72, 264, 8, 3), (1025, 136, 200, 64, 7), (3000, 512, 384, 32, 2), (1100, 2056, 72, 128, 2), (2000, 64, 128, 16, 700), (40, 104, 8, 56, 4096),
    (17000, 72, 136, 8, 3), (16500, 264, 72, 24, 5), (1600, 520, 1000, 56, 2), (1100, 136, 520, 120, 40), (12000, 328, 200, 48, 9),
])
def test_against_the_formula(tokens, dim, width, rank, adapters, dtype):
    x, y, a, b, scales, ids = make(tokens, dim, width, rank, adapters, dtype, seed=tokens + dim)
    want, off = exact(x, y, a, b, scales, ids)
    plan = ops.LoraPlan(ids, adapters)
    before = y.clone()
    out = torch.full_like(y, 77.0)
    assert ops.lora_add(y, x, ops.LoraAdapters(a, b, scales), plan, out=out) is out
    check(out, want, off, dtype)
    assert torch.equal(y, before) and torch.equal(out[ids < 0], y[ids < 0])
    assert ops.lora_add(y, x, ops.LoraAdapters(a, b, scales), plan) is y
    assert torch.equal(y, out)


# (each of the ways that a call can go: few tokens, several, and many by tiles times ranks)
@pytest.mark.parametrize("tokens,rank,adapters", [(50, 32, 6), (1500, 32, 6), (1500, 32, 120), (300, 128, 30), (1600, 64, 2), (1200, 24, 1), (20000, 16, 3), (1100, 128, 40)])
def test_ranks_and_what_lies_behind_them(tokens, rank, adapters):
    x, y, a, b, scales, ids = make(tokens, 264, 72, rank, adapters, bf16, seed=3)
    ranks = torch.tensor(([rank, 0, 1, 7, 16, rank - 2] * adapters)[:adapters], dtype=torch.int32)
    for n, r in enumerate(ranks.tolist()):
        a[n, r:] = float("nan")
        b[n, :, r:] = float("inf")
    want, off = exact(x, y, a, b, None, ids, ranks)
    got = ops.lora_add(y, x, ops.LoraAdapters(a, b, None, ranks.cuda()), ops.LoraPlan(ids, adapters), out=torch.empty_like(y))
    check(got, want, off, bf16)


@pytest.mark.parametrize("tokens,adapters", [(40, 4), (1300, 4), (1300, 250), (17000, 4)])
def test_views_leave_the_rest_alone(tokens, adapters):
    x, y, a, b, scales, ids = make(tokens, 128, 256, 16, adapters, bf16, seed=4)
    wide_x, wide_y = torch.full((tokens, 400), 3.0, dtype=bf16, device="cuda"), torch.full((tokens, 1000), 5.0, dtype=bf16, device="cuda")
    wide_x[:, 8:136], wide_y[:, 504:760] = x, y
    wide_a, wide_b = torch.full((adapters, 48, 136), float("nan"), dtype=bf16, device="cuda"), torch.full((adapters, 260, 48), float("nan"), dtype=bf16, device="cuda")
    wide_a[:, 16:32, :128], wide_b[:, 2:258, 8:24] = a, b
    want = ops.lora_add(y, x, ops.LoraAdapters(a, b, scales), ops.LoraPlan(ids, adapters), out=torch.empty_like(y))
    ops.lora_add(wide_y[:, 504:760], wide_x[:, 8:136], ops.LoraAdapters(wide_a[:, 16:32, :128], wide_b[:, 2:258, 8:24], scales), ops.LoraPlan(ids, adapters))
    assert torch.equal(wide_y[:, 504:760], want)
    assert (wide_y[:, :504] == 5.0).all() and (wide_y[:, 760:] == 5.0).all()


def test_one_tensor_read_and_written():
    x, _, a, b, scales, ids = make(90, 512, 512, 32, 3, bf16, seed=6)
    plan, adapters = ops.LoraPlan(ids, 3), ops.LoraAdapters(a, b, scales)
    want = ops.lora_add(x, x, adapters, plan, out=torch.empty_like(x))
    ops.lora_add(x, x, adapters, plan)
    assert torch.equal(x, want)


# (each way that a call can go, the last two in the kernel of many tokens, which otherwise has several clusters to a tile)
@pytest.mark.parametrize("y_too", [True, False])
@pytest.mark.parametrize("tokens,dim,width,rank,adapters", [(50, 512, 512, 32, 6), (1500, 512, 512, 32, 6), (3000, 1024, 1024, 128, 4), (3500, 1024, 2048, 128, 1), (1600, 512, 512, 64, 2)])
def test_x_in_the_place_of_out(tokens, dim, width, rank, adapters, y_too):
    x, y, a, b, scales, ids = make(tokens, dim, width, rank, adapters, bf16, seed=tokens)
    if y_too:
        y[:, :dim] = x
    want, off = exact(x, y, a, b, scales, ids)
    out = y if y_too else torch.zeros_like(y)
    out[:, :dim] = x
    ops.lora_add(y, out[:, :dim], ops.LoraAdapters(a, b, scales), ops.LoraPlan(ids, adapters), out=out)
    check(out, want, off, bf16)


@pytest.mark.parametrize("tokens,rank,adapters", [(70, 16, 2), (1100, 16, 2), (1100, 64, 50), (1500, 64, 2), (17000, 16, 2), (1100, 128, 40)])
@pytest.mark.parametrize("std", [2.0 ** -20, 1.0, 3000.0])
def test_half_precision_products_far_from_one(std, tokens, rank, adapters):
    x, y, a, b, scales, ids = make(tokens, 64, 64, rank, adapters, f16, seed=7, std=std)
    y, a = y * 0, a * 40  # (x A^T past fp16's largest number, or below its smallest)
    b = (b.float() * min(1.0, 1.0 / (std * 40))).to(f16)
    want, off = exact(x, y, a, b, scales, ids)
    check(ops.lora_add(y, x, ops.LoraAdapters(a, b, scales), ops.LoraPlan(ids, adapters)), want, off, f16)


@pytest.mark.parametrize("tokens,adapters", [(40, 2), (1200, 2), (1200, 230), (17000, 3)])
def test_infinities_of_one_token_stay_its_own(tokens, adapters):
    x, y, a, b, scales, ids = make(tokens, 64, 64, 16, adapters, bf16, seed=8)
    ids[:] = 1
    want, off = exact(x, y, a, b, scales, ids)
    x[3, 5], x[4, 6] = float("inf"), float("nan")
    got = ops.lora_add(y, x, ops.LoraAdapters(a, b, scales), ops.LoraPlan(ids, adapters), out=torch.empty_like(y))
    assert not got[3].isfinite().any() and got[4].isnan().all()
    rest = torch.tensor([i for i in range(tokens) if i not in (3, 4)], device="cuda")
    check(got[rest], want[rest], off[rest], bf16)
    # one rank: an infinity stays an infinity
    a1, b1 = a[:, :8].clone(), b[:, :, :8].clone()
    got = ops.lora_add(y, x, ops.LoraAdapters(a1, b1, scales, torch.ones(adapters, dtype=torch.int32, device="cuda")), ops.LoraPlan(ids, adapters), out=torch.empty_like(y))
    assert torch.equal(got[3].float(), float("inf") * (torch.sign(a1[1, 0, 5]) * torch.sign(b1[1, :, 0])).float())


def test_rows_behind_the_last_and_two_streams_at_once():
    # Calls of every way on two streams; each has its own workspace, and what lies behind the tokens stays as it was.
    made = []
    for seed, (tokens, rank, adapters) in enumerate([(60, 16, 3), (1300, 32, 3), (1300, 64, 60), (1300, 128, 3), (1100, 128, 40)] * 2):
        x, y, a, b, scales, ids = make(tokens, 256, 320, rank, adapters, bf16, seed=20 + seed)
        out = torch.full((tokens + 40, 320), 7.0, dtype=bf16, device="cuda")
        made.append((x, y, ops.LoraAdapters(a, b, scales), ops.LoraPlan(ids, adapters), out, exact(x, y, a, b, scales, ids), tokens))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, (x, y, adapters, plan, out, _, tokens) in enumerate(made):
            with torch.cuda.stream(streams[i % 2]):
                ops.lora_add(y, x, adapters, plan, out=out[:tokens])
    torch.cuda.synchronize()
    for _, _, _, _, out, (want, off), tokens in made:
        check(out[:tokens], want, off, bf16)
        assert (out[tokens:] == 7.0).all()


@pytest.mark.parametrize("tokens", [30, 1200, 17000])
def test_adapters_and_ranks_outside_raise_a_bit(tokens):
    x, y, a, b, scales, ids = make(tokens, 64, 64, 16, 3, bf16, seed=9)
    plan = ops.LoraPlan(ids, 3)
    want = ops.lora_add(y, x, ops.LoraAdapters(a, b, scales), plan, out=torch.empty_like(y))
    wrong = torch.where(ids < 0, 3 + torch.arange(tokens, dtype=torch.int32, device="cuda") * 1000000, ids)
    got = ops.lora_add(y, x, ops.LoraAdapters(a, b, scales), ops.LoraPlan(wrong, 3), out=torch.empty_like(y))
    assert torch.equal(got, want) and ops.lora_status(clear=True) == 1
    ranks = torch.tensor([17, 16, 1 << 30], dtype=torch.int32, device="cuda")
    got = ops.lora_add(y, x, ops.LoraAdapters(a, b, scales, ranks), plan, out=torch.empty_like(y))
    assert torch.equal(got, want) and ops.lora_status(clear=True) == 2
    ops.lora_add(y, x, ops.LoraAdapters(a, b, scales, torch.full((3,), -5, dtype=torch.int32, device="cuda")), plan)
    assert ops.lora_status(clear=True) == 2


@pytest.mark.parametrize("tokens,rank,adapters", [(33, 16, 3), (1600, 64, 3), (1100, 128, 40)])
def test_nobody_has_an_adapter_and_no_tokens(tokens, rank, adapters):
    x, y, a, b, scales, ids = make(tokens, 64, 64, rank, adapters, bf16, seed=10)
    ids[:] = -1
    out = ops.lora_add(y, x, ops.LoraAdapters(a, b, scales), ops.LoraPlan(ids, adapters), out=torch.empty_like(y))
    assert torch.equal(out, y)
    none = ops.LoraPlan(ids[:0], adapters)
    assert ops.lora_add(y[:0], x[:0], ops.LoraAdapters(a, b, scales), none).shape == (0, 64)


@pytest.mark.parametrize("tokens,rank,n", [(48, 16, 5), (1600, 64, 2), (1100, 128, 40)])
def test_a_captured_step_with_its_plan(tokens, rank, n):
    x, y, a, b, scales, ids = make(tokens, 512, 512, rank, n, bf16, seed=11)
    adapters, out = ops.LoraAdapters(a, b, scales), torch.empty_like(y)
    changing = ids.clone()
    plan = ops.LoraPlan(changing, n)
    ops.lora_add(y, x, adapters, plan, out=out)
    graph, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=s):
        plan.fill()
        ops.lora_add(y, x, adapters, plan, out=out)
        second = ops.lora_add(out, x, adapters, plan, out=torch.empty_like(y))
    for shift in range(3):
        changing.copy_((ids + shift) % n - (ids + shift) % 2)
        graph.replay()
        torch.cuda.synchronize()
        want, off = exact(x, y, a, b, scales, changing)
        check(out, want, off, bf16)
        want, off = exact(x, out, a, b, scales, changing)
        check(second, want, off, bf16)


@pytest.mark.parametrize("tokens,rank,adapters", [(300, 32, 20), (1600, 64, 2), (1100, 128, 40)])
def test_the_same_call_gives_the_same_bits(tokens, rank, adapters):
    x, y, a, b, scales, ids = make(tokens, 1032, 520, rank, adapters, bf16, seed=12)
    plan, adapters = ops.LoraPlan(ids, adapters), ops.LoraAdapters(a, b, scales)
    first = ops.lora_add(y, x, adapters, plan, out=torch.empty_like(y))
    for _ in range(20):
        assert torch.equal(ops.lora_add(y, x, adapters, plan, out=torch.empty_like(y)), first)
