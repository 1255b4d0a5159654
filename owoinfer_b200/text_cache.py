"""The paged caches of a text decoder's layers, and a small decoder that writes with them: `python -m owoinfer_b200.text_cache`.

The image model's rows of text come from a language model that reads a prompt and may rewrite it first. `TextCache` keeps what its
layers need between calls: per layer a pool of pages, for the batch one block table, lengths and positions. `Decoder` is a plain
decoder of random weights whose layers run qk_norm_rope_append, attention_paged for a prompt, attention_paged_decode for every
word after it and, where the caches are to stay within a budget, kv_evict; products with weights are library matrix products."""
import argparse

import torch

from . import ops


def rope_table(positions, dim, base=1e6, device="cuda"):
    """fp32 [positions, dim]: sin | cos of the dim / 2 angles of each position."""
    inv = base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    angles = torch.arange(positions, dtype=torch.float64)[:, None] * inv
    return torch.cat([angles.sin(), angles.cos()], 1).float().contiguous().to(device)


class TextCache:
    """Pages of `layers` caches for `batch` sequences of up to `slots` slots. With a budget a cache that is full shrinks to it: the first
    `sinks` slots, the last `recent` and of the rest those of most weight stay, for each layer and key head by itself; the
    sequences keep counting positions. What stays moves to a second set of pages, which takes turns with the first. Weights are those that the
    tokens written one by one gave; a prompt's own attention is not counted, so that of slots without any weight yet the lowest stay."""

    def __init__(self, layers, batch, kv_heads, head_dim, slots, page_size=64, budget=0, sinks=4, recent=0, dtype=torch.bfloat16, device="cuda"):
        width = -(-slots // page_size)
        self.slots, self.budget, self.sinks, self.recent = width * page_size, budget, sinks, recent
        if budget and not sinks + recent <= budget < self.slots:
            raise ValueError("the budget must hold the sinks and the recent slots and be below the slots")
        sets = 2 if budget else 1
        shape = (layers, sets * batch * width, kv_heads, page_size, head_dim)
        self.k, self.v = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
        pages = torch.arange(sets * batch * width, dtype=torch.int32, device=device).view(sets, batch, width)
        self.tables, self.used = list(pages.unbind(0)), 0
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self.positions = torch.zeros(batch, dtype=torch.int32, device=device)  # of the next token
        self.each = torch.arange(batch + 1, dtype=torch.int32, device=device)  # cu_seqlens of a token each
        self.weights = [torch.zeros((layers, batch, kv_heads, self.slots), device=device) for _ in range(sets)] if budget else None
        self.longest = 0  # no sequence is longer, as far as the host knows
        self._views()

    def _views(self):
        self.layers = [ops.PagedCache(k, v, self.tables[self.used], self.lens) for k, v in zip(self.k, self.v)]

    def grow(self, tokens):
        """Makes room for tokens[b] more of each sequence (a list), or for one more of each (None)."""
        most = 1 if tokens is None else max(tokens)
        if self.longest + most > self.slots and self.budget and self.longest > self.budget:
            self.evict()
        if self.longest + most > self.slots:
            raise ValueError("the cache is full")
        more = 1 if tokens is None else torch.tensor(tokens, dtype=torch.int32, device=self.lens.device)
        self.lens += more
        self.positions += more
        self.longest += most

    def evict(self):
        """Every cache to its budget, in the other set of pages."""
        other = 1 - self.used
        lens = torch.empty_like(self.lens)  # (every layer's call writes the same)
        for i, cache in enumerate(self.layers):
            ops.kv_evict(cache, self.weights[self.used][i], self.tables[other], self.budget, sinks=self.sinks, recent=self.recent, lens_out=lens,
                         weights_out=self.weights[other][i])
        self.lens, self.used, self.longest = lens, other, min(self.longest, self.budget)
        self._views()


class Decoder:
    """Layers of norm, attention with per-head norms and rotation, norm, gated feed-forward; random weights from a seed."""

    def __init__(self, vocab=512, dim=512, layers=2, q_heads=8, kv_heads=2, head_dim=64, positions=8192, window=0, sinks=0, seed=0,
                 dtype=torch.bfloat16, device="cuda"):
        g = torch.Generator().manual_seed(seed)
        w = lambda *shape: (torch.randn(shape, generator=g) * shape[-1] ** -0.5).to(device, dtype)  # noqa: E731
        self.kv_heads, self.head_dim, self.dtype, self.window, self.sinks = kv_heads, head_dim, dtype, window, sinks
        self.scale = head_dim ** -0.5
        self.rope = rope_table(positions, head_dim, device=device)
        self.embedding = w(vocab, dim)
        self.layers = [dict(qkv=w((q_heads + 2 * kv_heads) * head_dim, dim), out=w(dim, q_heads * head_dim), up=w(4 * dim, dim), down=w(dim, 2 * dim),
                            q_norm=1 + w(head_dim) * 0.1, k_norm=1 + w(head_dim) * 0.1) for _ in range(layers)]

    def cache(self, batch, slots, **how):
        return TextCache(len(self.layers), batch, self.kv_heads, self.head_dim, slots, dtype=self.dtype, device=self.rope.device, **how)

    def _norm(self, x):
        return (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)).to(self.dtype)

    def _run(self, x, cache, cu, positions, attention):
        for i, (w, paged) in enumerate(zip(self.layers, cache.layers)):
            q = ops.qk_norm_rope_append(self._norm(x) @ w["qkv"].T, paged, cu, w["q_norm"], w["k_norm"], self.rope, positions=positions)
            out, _ = attention(i, q, paged)
            x = x + out.flatten(1) @ w["out"].T
            gate, up = (self._norm(x) @ w["up"].T).chunk(2, -1)
            x = x + (torch.nn.functional.silu(gate) * up) @ w["down"].T
        return x

    def _logits(self, x):
        return self._norm(x) @ self.embedding.T

    def read(self, prompts, cache):
        """Prompts (lists of token numbers, none empty) into an empty cache: the logits after each one's last token."""
        counts = [len(p) for p in prompts]
        if min(counts) == 0 or cache.longest:
            raise ValueError("read takes prompts of a token at least, and an empty cache")
        device = self.rope.device
        cache.grow(counts)
        cu = torch.tensor([0] + counts).cumsum(0).to(device, torch.int32)
        x = self.embedding[torch.tensor(sum(prompts, []), device=device)].float()
        x = self._run(x, cache, cu, None,
                      lambda i, q, paged: ops.attention_paged(q, paged, cu, max(counts), self.scale, self.window, self.sinks))
        return self._logits(x[cu[1:].long() - 1])

    def write(self, tokens, cache):
        """One token more of every sequence (a tensor [batch]): the logits after it."""
        cache.grow(None)
        weights = None if cache.weights is None else cache.weights[cache.used]
        x = self._run(self.embedding[tokens].float(), cache, cache.each, cache.positions - 1,
                      lambda i, q, paged: ops.attention_paged_decode(q, paged, self.scale, cache.longest, self.window, self.sinks,
                                                                     weights=None if weights is None else weights[i]))
        return self._logits(x)


def main(argv=None):
    p = argparse.ArgumentParser(prog="python -m owoinfer_b200.text_cache", description="Greedy words of a small random decoder over paged caches.")
    p.add_argument("--prompts", type=int, nargs="+", default=[40, 7, 131], help="tokens of each prompt")
    p.add_argument("--words", type=int, default=200, help="tokens to write after each")
    p.add_argument("--slots", type=int, default=256, help="slots of a sequence's cache")
    p.add_argument("--budget", type=int, default=128, help="slots that a full cache shrinks to (0: it never does)")
    a = p.parse_args(argv)
    model = Decoder(positions=max(a.prompts) + a.words + 1)
    cache = model.cache(len(a.prompts), a.slots, budget=a.budget, sinks=4, recent=a.budget // 4)
    g = torch.Generator().manual_seed(1)
    logits = model.read([torch.randint(len(model.embedding), (n,), generator=g).tolist() for n in a.prompts], cache)
    words, shrunk = [], 0
    for _ in range(a.words):
        words.append(logits.argmax(-1))
        used = cache.used
        logits = model.write(words[-1], cache)
        shrunk += cache.used != used
    for n, row in zip(a.prompts, torch.stack(words, 1).tolist()):
        print(f"prompt of {n}: {row[:12]} ... {row[-4:]}")
    print(f"caches hold {cache.lens.tolist()} slots at positions {cache.positions.tolist()}, shrunk {shrunk} times; status {ops.paged_cache_status()}")


if __name__ == "__main__":
    main()
