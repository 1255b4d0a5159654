"""The paged caches of a text decoder's layers, and a small decoder that writes with them: `python -m owoinfer_b200.text_cache`.

The image model's rows of text come from a language model that reads a prompt and may rewrite it first. `TextCache` keeps what its
layers need between calls: per layer a pool of pages, for the batch one block table, lengths and positions. `Decoder` is a plain
decoder of random weights whose layers run qk_norm_rope_append, attention_paged for a prompt, attention_paged_decode for every
word after it and, where the caches are to stay within a budget, kv_evict; products with weights are library matrix products. With 8 bits
the projections behind a norm are int8_gemm on what add_rms_norm_quantize makes of the residual stream; with adapters every request may
have a low-rank one beside all projections (lora_add); token_logprobs says how probable a text is, or what else could follow."""
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


def quantize_rows(w):
    """(int8 [n, k], fp32 [n]): a weight in 8 bits with a scale for each row, as int8_gemm takes it."""
    scale = (w.float().abs().amax(1) / 127.0).clamp(min=1e-30)
    return (w.float() / scale[:, None]).round().to(torch.int8).contiguous(), scale


class Decoder:
    """Layers of norm, attention with per-head norms and rotation, norm, gated feed-forward; random weights from a seed. bits 8: the two
    projections behind a norm in INT8 (bf16 only). adapters: low-rank adapters of `rank` beside all four projections; which request has
    which is the plan that read, write and score take."""

    def __init__(self, vocab=512, dim=512, layers=2, q_heads=8, kv_heads=2, head_dim=64, positions=8192, window=0, sinks=0, seed=0,
                 dtype=torch.bfloat16, device="cuda", bits=16, adapters=0, rank=16):
        if bits not in (8, 16) or (bits == 8 and dtype != torch.bfloat16):
            raise ValueError("bits must be 16, or 8 with bf16")
        g = torch.Generator().manual_seed(seed)
        w = lambda *shape: (torch.randn(shape, generator=g) * shape[-1] ** -0.5).to(device, dtype)  # noqa: E731
        self.kv_heads, self.head_dim, self.dtype, self.window, self.sinks = kv_heads, head_dim, dtype, window, sinks
        self.scale = head_dim ** -0.5
        self.rope = rope_table(positions, head_dim, device=device)
        self.embedding = w(vocab, dim)
        self.layers = [dict(qkv=w((q_heads + 2 * kv_heads) * head_dim, dim), out=w(dim, q_heads * head_dim), up=w(4 * dim, dim), down=w(dim, 2 * dim),
                            q_norm=1 + w(head_dim) * 0.1, k_norm=1 + w(head_dim) * 0.1) for _ in range(layers)]
        self.bits, self.adapters, self.rank = bits, adapters, rank
        if bits == 8:
            for layer in self.layers:
                layer["qkv"], layer["up"] = quantize_rows(layer["qkv"]), quantize_rows(layer["up"])
        if adapters:
            scales = torch.full((adapters,), 0.5, device=device)
            shapes = dict(qkv=((q_heads + 2 * kv_heads) * head_dim, dim), out=(dim, q_heads * head_dim), up=(4 * dim, dim), down=(dim, 2 * dim))
            for layer in self.layers:
                layer["adapters"] = {name: ops.LoraAdapters(w(adapters, rank, k), w(adapters, n, rank), scales) for name, (n, k) in shapes.items()}

    def cache(self, batch, slots, **how):
        return TextCache(len(self.layers), batch, self.kv_heads, self.head_dim, slots, dtype=self.dtype, device=self.rope.device, **how)

    def _norm(self, x):
        return (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)).to(self.dtype)

    def plan(self, adapters, counts=None):
        """The plan of a pass in which request i has counts[i] tokens (None: one each) and the adapter adapters[i] (-1: none)."""
        each = torch.tensor(adapters, dtype=torch.int32)
        if counts is not None:
            each = each.repeat_interleave(torch.tensor(counts))
        return ops.LoraPlan(each.to(self.rope.device), self.adapters)

    def _project(self, w, name, x, plan):
        y = x @ w[name].T
        return y if plan is None else ops.lora_add(y, x, w["adapters"][name], plan)

    def _project_norm(self, w, name, stream, more, plan):
        """The projection of the norm of stream + more (None: nothing), and that sum: in the stream's place with 8 bits."""
        if self.bits == 16:
            stream = stream if more is None else stream + more
            return self._project(w, name, self._norm(stream), plan), stream
        norm = None if plan is None else torch.empty(stream.shape, dtype=self.dtype, device=stream.device)
        if more is None:
            q, scale = ops.add_rms_norm_quantize(stream, norm_out=norm)
        else:
            q, scale = ops.add_rms_norm_quantize(more, residual=stream, norm_out=norm)
        y = ops.int8_gemm(q, scale, *w[name])
        return (y if plan is None else ops.lora_add(y, norm, w["adapters"][name], plan)), stream

    def _run(self, x, cache, cu, positions, attention, plan=None):
        more = None  # what the layer before has left to be added
        for i, (w, paged) in enumerate(zip(self.layers, cache.layers)):
            qkv, x = self._project_norm(w, "qkv", x, more, plan)
            q = ops.qk_norm_rope_append(qkv, paged, cu, w["q_norm"], w["k_norm"], self.rope, positions=positions)
            out, _ = attention(i, q, paged)
            up, x = self._project_norm(w, "up", x, self._project(w, "out", out.flatten(1), plan), plan)
            gate, up = up.chunk(2, -1)
            more = self._project(w, "down", torch.nn.functional.silu(gate) * up, plan)
        return x if more is None else x + more

    def _logits(self, x):
        return self._norm(x) @ self.embedding.T

    def _read(self, prompts, cache, plan):
        counts = [len(p) for p in prompts]
        if min(counts) == 0 or cache.longest:
            raise ValueError("read takes prompts of a token at least, and an empty cache")
        device = self.rope.device
        cache.grow(counts)
        cu = torch.tensor([0] + counts).cumsum(0).to(device, torch.int32)
        x = self.embedding[torch.tensor(sum(prompts, []), device=device)].float()
        x = self._run(x, cache, cu, None,
                      lambda i, q, paged: ops.attention_paged(q, paged, cu, max(counts), self.scale, self.window, self.sinks), plan)
        return x, cu[1:].long() - 1

    def read(self, prompts, cache, plan=None):
        """Prompts (lists of token numbers, none empty) into an empty cache: the logits after each one's last token."""
        x, last = self._read(prompts, cache, plan)
        return self._logits(x[last])

    def score(self, prompts, cache, plan=None, top=0):
        """Prompts into an empty cache, as read: TokenLogprobs of each token's successor in its prompt (none behind the last), with the entropy
        and the `top` most probable tokens in its place."""
        x, last = self._read(prompts, cache, plan)
        targets = torch.tensor(sum(prompts, []), device=x.device).roll(-1)
        targets[last] = -1
        return ops.token_logprobs(self._logits(x), targets, top=top)

    def write(self, tokens, cache, plan=None):
        """One token more of every sequence (a tensor [batch]): the logits after it."""
        cache.grow(None)
        weights = None if cache.weights is None else cache.weights[cache.used]
        x = self._run(self.embedding[tokens].float(), cache, cache.each, cache.positions - 1,
                      lambda i, q, paged: ops.attention_paged_decode(q, paged, self.scale, cache.longest, self.window, self.sinks,
                                                                     weights=None if weights is None else weights[i]), plan)
        return self._logits(x)


def main(argv=None):
    p = argparse.ArgumentParser(prog="python -m owoinfer_b200.text_cache", description="Greedy words of a small random decoder over paged caches.")
    p.add_argument("--prompts", type=int, nargs="+", default=[40, 7, 131], help="tokens of each prompt")
    p.add_argument("--words", type=int, default=200, help="tokens to write after each")
    p.add_argument("--slots", type=int, default=256, help="slots of a sequence's cache")
    p.add_argument("--budget", type=int, default=128, help="slots that a full cache shrinks to (0: it never does)")
    p.add_argument("--int8", action="store_true", help="the projections behind a norm in INT8")
    p.add_argument("--adapters", type=int, default=0, help="adapters, which the prompts have in turn, every other prompt none (0: nobody has one)")
    p.add_argument("--top", type=int, default=0, help="of the last word: so many of the most probable ones, with their probabilities")
    a = p.parse_args(argv)
    model = Decoder(positions=max(a.prompts) + a.words + 1, bits=8 if a.int8 else 16, adapters=a.adapters)
    who = [i // 2 % a.adapters if i % 2 == 0 else -1 for i in range(len(a.prompts))] if a.adapters else None
    plan = model.plan(who) if who else None
    cache = model.cache(len(a.prompts), a.slots, budget=a.budget, sinks=4, recent=a.budget // 4)
    g = torch.Generator().manual_seed(1)
    logits = model.read([torch.randint(len(model.embedding), (n,), generator=g).tolist() for n in a.prompts], cache, model.plan(who, a.prompts) if who else None)
    words, shrunk = [], 0
    for _ in range(a.words):
        words.append(logits.argmax(-1))
        said = ops.token_logprobs(logits, words[-1], top=a.top) if a.top else None
        used = cache.used
        logits = model.write(words[-1], cache, plan)
        shrunk += cache.used != used
    for n, row in zip(a.prompts, torch.stack(words, 1).tolist()):
        print(f"prompt of {n}: {row[:12]} ... {row[-4:]}")
    if a.top and words:
        for n, mine, tokens, others in zip(a.prompts, said.logprobs.exp().tolist(), said.top_tokens.tolist(), said.top_logprobs.exp().tolist()):
            print(f"prompt of {n}: the last word has probability {mine:.3f}; most probable " + ", ".join(f"{t} {q:.3f}" for t, q in zip(tokens, others)))
    print(f"caches hold {cache.lens.tolist()} slots at positions {cache.positions.tolist()}, shrunk {shrunk} times; status {ops.paged_cache_status()}")


if __name__ == "__main__":
    main()
