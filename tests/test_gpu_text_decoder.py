"""The operators around a decoder's attention as its steps run them: in INT8, with adapters, its log probabilities."""
import pytest
import torch

from owoinfer_b200 import ops
from owoinfer_b200.text_cache import Decoder, main, quantize_rows

pytestmark = pytest.mark.gpu
bf16 = torch.bfloat16


@pytest.fixture(autouse=True)
def _status():
    ops.lora_status(clear=True), ops.paged_cache_status(clear=True)
    yield
    assert ops.lora_status(clear=True) == 0 and ops.paged_cache_status(clear=True) == 0 and ops.kernel_status() == (0, 0)


def prompts(counts, vocab=512, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(vocab, (n,), generator=g).tolist() for n in counts]


def text(model, texts, who=None, words=3):
    """The logits after the prompts and after each of some words."""
    counts = [len(p) for p in texts]
    cache = model.cache(len(texts), max(counts) + words)
    got = [model.read(texts, cache, None if who is None else model.plan(who, counts))]
    plan = None if who is None else model.plan(who)
    for i in range(words):
        got.append(model.write(torch.arange(len(texts), device="cuda") * 7 + i, cache, plan))
    return got


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("counts", [[40, 7, 131, 1], [300, 250, 2, 90]])
def test_every_sequence_has_its_own_adapter(bits, counts):
    model = Decoder(bits=bits, adapters=3)
    texts = prompts(counts)
    who = [2, -1, 0, 2]
    mixed = text(model, texts, who)
    for adapter in (-1, 0, 2):
        alone = text(model, texts, [adapter] * 4)
        for a, b in zip(mixed, alone):
            for i in range(4):
                if who[i] == adapter:
                    assert torch.equal(a[i], b[i])
    assert not torch.equal(mixed[0][0], text(model, texts, [-1] * 4, words=0)[0][0])


@pytest.mark.parametrize("bits", [16, 8])
def test_nobody_has_an_adapter(bits):
    model = Decoder(bits=bits, adapters=3)
    texts = prompts([40, 7, 131])
    for a, b in zip(text(model, texts), text(model, texts, [-1, -1, -1])):
        assert torch.equal(a, b)


def test_score_and_logits_say_the_same():
    model = Decoder(bits=8)
    texts = prompts([20, 1, 64])
    said = model.score(texts, model.cache(3, 64), top=4)
    x, last = model._read(texts, model.cache(3, 64), None)
    want = torch.log_softmax(model._logits(x).double(), -1)
    start = 0
    for p in texts:
        for i, token in enumerate(p[1:]):
            # The sum of 512 exponentials is off by at most 512 roundings of 2^-24 (3.1e-5), the logarithm and the logit (below 16) by 1e-6.
            assert abs(float(said.logprobs[start + i]) - float(want[start + i, token])) < 1e-4
        assert said.logprobs[start + len(p) - 1] == 0 and said.ranks[start + len(p) - 1] == 0
        start += len(p)
    assert torch.equal(said.top_tokens[:, 0].long(), want.argmax(-1))


@pytest.mark.parametrize("tokens", [1, 33, 400])
def test_a_step_together_eager_and_captured(tokens):
    # Stream + output -> norm -> INT8 projection + adapters -> log probabilities, against 64 bits from the codes on.
    dim, width, n = 512, 1032, 4
    g = torch.Generator(device="cuda").manual_seed(tokens)
    r = lambda *shape, s=1.0: s * torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    stream, more, weight = r(tokens, dim, s=3.0), r(tokens, dim).to(bf16), (1 + r(dim, s=0.1)).to(bf16)
    w8, ws = quantize_rows(r(width, dim, s=dim ** -0.5))
    adapters = ops.LoraAdapters(r(n, 16, dim, s=dim ** -0.5).to(bf16), r(n, width, 16, s=0.25).to(bf16))
    ids = torch.arange(tokens, dtype=torch.int32, device="cuda") % (n + 1) - 1
    targets = torch.arange(tokens, device="cuda") % width
    plan = ops.LoraPlan(ids, n)

    def step():
        total, norm = torch.empty_like(stream), torch.empty(tokens, dim, dtype=bf16, device="cuda")
        q, scale = ops.add_rms_norm_quantize(more, weight, stream, residual_out=total, norm_out=norm)
        y = ops.lora_add(ops.int8_gemm(q, scale, w8, ws), norm, adapters, plan)
        return (total, norm, q, scale, y) + tuple(ops.token_logprobs(y, targets, top=3))

    want = step()
    total, norm, q, scale, y = want[:5]
    s = stream.double() + more.double()
    exact = s / (s.square().mean(-1, keepdim=True) + 1e-6).sqrt() * weight.double()
    # A code is off by half a step, so a product by half a step times the sum of the weights; 1e-5 of it for the fp32 on the way.
    w = w8.double() * ws.double()[:, None]
    out = exact @ w.T
    off = (scale.double()[:, None] / 2 + 1e-5 * exact.abs().amax(-1, keepdim=True)) * w.abs().sum(1)
    for t in range(tokens):
        if ids[t] >= 0:
            a, b = adapters.a[ids[t]].double(), adapters.b[ids[t]].double()
            out[t] += (norm[t].double() @ a.T) @ b.T
            off[t] += 2.0 ** -12 * ((norm[t].double().abs() @ a.abs().T) @ b.abs().T)
    half = torch.finfo(bf16).eps / 2
    # Rounded to bf16 by the projection and once more behind the adapters, each by half a step of what it holds.
    first = (exact @ w.T).abs() + off
    assert ((y.double() - out).abs() <= off + first * half * 1.01 + (out.abs() + off) * half * 1.01).all()

    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        got = step()
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_refusals():
    with pytest.raises(ValueError, match="bits"):
        Decoder(bits=4)
    with pytest.raises(ValueError, match="bits"):
        Decoder(bits=8, dtype=torch.float16)


def test_the_command(capsys):
    main(["--prompts", "30", "5", "9", "--words", "40", "--slots", "64", "--budget", "32", "--int8", "--adapters", "2", "--top", "3"])
    out = capsys.readouterr().out
    assert out.count("prompt of") == 6 and "most probable" in out and "status 0" in out
