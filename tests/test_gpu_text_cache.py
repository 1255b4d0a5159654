"""A small decoder over paged caches against the same decoder with plain attention in 64 bits, and with caches that shrink."""
import pytest
import torch

pytestmark = pytest.mark.gpu

# A layer's two additions to a row pass about ten roundings to 8 bits (norm, product, rotated heads, attention, product; norm, product,
# gate, product), each off by 2^-9 of its value at most: two layers and the logits' own norm and product stay below 22 * 2^-9.
BOUND = 22 * 2.0 ** -9


def plain_logits(model, tokens):
    """Logits after every token of one sequence: the decoder's formulas in 64 bits."""
    d = torch.float64
    norm = lambda x: x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)  # noqa: E731
    n, dim = len(tokens), model.head_dim
    sin, cos = model.rope[:n].to(d)[:, None].chunk(2, -1)
    turn = lambda x: torch.cat([x[..., :dim // 2] * cos - x[..., dim // 2:] * sin, x[..., dim // 2:] * cos + x[..., :dim // 2] * sin], -1)  # noqa: E731
    at = torch.arange(n, device=model.rope.device)
    seen = at[None] <= at[:, None]
    if model.window:
        seen &= (at[:, None] - at[None] < model.window) | (at[None] < model.sinks)
    x = model.embedding[tokens].to(d)
    for w in model.layers:
        w = {k: t.to(d) for k, t in w.items()}
        qkv = (norm(x) @ w["qkv"].T).view(n, -1, dim)
        heads = qkv.shape[1] - 2 * model.kv_heads
        q, k, v = qkv.split([heads, model.kv_heads, model.kv_heads], 1)
        q, k = turn(norm(q) * w["q_norm"]), turn(norm(k) * w["k_norm"])
        k, v = (t.repeat_interleave(heads // model.kv_heads, 1) for t in (k, v))
        s = torch.einsum("ihd,jhd->hij", q, k) * model.scale
        p = s.masked_fill(~seen, -torch.inf).softmax(-1)
        x = x + torch.einsum("hij,jhd->ihd", p, v).flatten(1) @ w["out"].T
        gate, up = (norm(x) @ w["up"].T).chunk(2, -1)
        x = x + (torch.nn.functional.silu(gate) * up) @ w["down"].T
    return norm(x) @ model.embedding.to(d).T


def written(model, cache, prompts, words):
    """Logits after each prompt and after each of the given words [batch, n] behind them: [batch, n + 1, vocab]."""
    logits = [model.read(prompts, cache)]
    logits += [model.write(words[:, i], cache) for i in range(words.shape[1])]
    return torch.stack(logits, 1)


def setup(window=0, sinks=0, **how):
    from owoinfer_b200 import text_cache
    model = text_cache.Decoder(positions=512, window=window, sinks=sinks, **how)
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(512, (n,), generator=g).tolist() for n in (33, 1, 150)]
    words = torch.randint(512, (3, 60), generator=g).cuda()
    return model, prompts, words


def off(got, want):
    return ((got.double() - want).norm(dim=-1) / want.norm(dim=-1)).max().item()


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 4)])
@pytest.mark.parametrize("q_heads,kv_heads,head_dim", [(8, 2, 64), (4, 4, 128)])
def test_decoder_against_plain(window, sinks, q_heads, kv_heads, head_dim):
    from owoinfer_b200 import ops
    model, prompts, words = setup(window, sinks, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim)
    ops.paged_cache_status(clear=True)
    got = written(model, model.cache(3, 256), prompts, words)
    for b, prompt in enumerate(prompts):
        want = plain_logits(model, torch.tensor(prompt + words[b].tolist(), device="cuda"))[len(prompt) - 1:]
        assert off(got[b], want) < BOUND
    assert ops.paged_cache_status() == 0


def test_shrinking_within_a_window_changes_nothing():
    """With a window, a cache that keeps the sinks and as many slots as the window has holds all that is ever looked at."""
    from owoinfer_b200 import ops
    model, prompts, words = setup(window=40, sinks=4)
    cache = model.cache(3, 160, page_size=16, budget=44 + 3, sinks=4, recent=43)
    got = written(model, cache, prompts, words)
    want = written(model, model.cache(3, 256), prompts, words)
    assert cache.longest < 160 and cache.lens.tolist() != cache.positions.tolist()  # it did shrink
    assert off(got, want.double()) < BOUND
    assert ops.paged_cache_status() == 0


def test_shrinking_by_weight():
    from owoinfer_b200 import ops
    model, prompts, words = setup()
    cache = model.cache(3, 160, page_size=16, budget=100, sinks=4, recent=20)
    got = written(model, cache, prompts, words)
    assert torch.isfinite(got).all()
    # The longest starts at 150: full after 10 words, down to 100, and 50 words more.
    assert cache.positions.tolist() == [93, 61, 210] and cache.lens.max().item() <= 160
    for weights, paged in zip(cache.weights[cache.used], cache.layers):
        for b, n in enumerate(cache.lens.tolist()):
            assert torch.isfinite(weights[b, :, :n]).all() and (weights[b, :, :n] >= 0).all()
            assert (weights[b, :, n - 1] <= 4 * (1 + 1e-5)).all()  # the newest slot: at most 1 of each of its four query heads
    assert ops.paged_cache_status() == 0


def test_refusals():
    from owoinfer_b200 import text_cache
    model, prompts, words = setup()
    cache = model.cache(1, 16, page_size=16)
    with pytest.raises(ValueError, match="token at least"):
        model.read([[]], cache)
    model.read([list(range(16))], cache)
    with pytest.raises(ValueError, match="empty cache"):
        model.read([[1]], cache)
    with pytest.raises(ValueError, match="full"):
        model.write(words[:1, 0], cache)
    with pytest.raises(ValueError, match="budget"):
        text_cache.TextCache(1, 1, 1, 64, 64, budget=64)


def test_command(capsys):
    from owoinfer_b200 import text_cache
    text_cache.main(["--prompts", "20", "3", "--words", "50", "--slots", "64", "--budget", "32"])
    out = capsys.readouterr().out
    assert "positions [70, 53]" in out and "status 0" in out
