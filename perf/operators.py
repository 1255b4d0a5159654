"""The calls a language model's layer makes on a paged key-value cache, over the sizes a text side of this framework meets.

The language model in front of the image model (it writes or rewrites a prompt, then its hidden states are the text rows of the
denoising step) runs one such layer after the other; every layer has its cache. The kinds:

  append   ops.qk_norm_rope_append: norms of queries and keys per head, position rotation, keys and values into the cache's pages
  prompt   ops.attention_paged: attention of a prompt's tokens (or a chunk of them) over the cache, causal, with or without a
           sliding window that leaves a few first tokens visible
  decode   ops.attention_paged_decode: attention of one new token of each sequence, which also adds up what weight each cached
           token got
  evict    ops.kv_evict: a cache that has grown past its budget keeps its first tokens, its last ones and those of most weight

A cache is a pool of pages [pages, kv_heads, page, head_dim]; a sequence's slots are its pages in the order of its row of the block
table. The plain forms below gather the pages, compute in 32 bits and round once.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
ROPE_BASE = 1e6
EPS = 1e-6


def _case(kind, batch, q_heads, kv_heads, head_dim, page, dtype="bf16", new=1, past=0, ragged=True, empty=False, window=0, sinks=0,
          rot=0, interleaved=False, shift=0, budget=0, recent=0):
    """new: tokens of the call of the longest sequence; past: tokens its cache holds ahead of them. ragged: the other sequences are
    shorter; empty: the last one has nothing at all. rot: rotated channels (0: all); shift: a token's position minus its slot."""
    return {"kind": kind, "batch": batch, "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "dtype": dtype,
            "new": new, "past": past, "ragged": ragged, "empty": empty, "window": window, "sinks": sinks, "rot": rot,
            "interleaved": interleaved, "shift": shift, "budget": budget, "recent": recent}


def listed():
    named = {
        # One sequence, one token: what every layer does between two words of a prompt that is being written. Latency alone.
        "append one token": _case("append", 1, 16, 8, 128, 16, past=700),
        # A batch of users, a token each, after evictions (positions run ahead of the slots), half of the channels rotated.
        "append 96 tokens": _case("append", 96, 32, 4, 128, 64, past=1500, rot=64, interleaved=True, shift=911),
        # Several prompts in one pass, of uneven lengths.
        "append prompts": _case("append", 7, 32, 8, 128, 64, new=4096),
        # Short prompts, the everyday text of an image: one pass over a ragged batch, no cache ahead of them.
        "prompts 300": _case("prompt", 5, 16, 8, 128, 16, new=297),
        # A chunk of a long prompt over what the cache holds already; narrow heads, a group of seven, half precision.
        "chunk 509 of 8k": _case("prompt", 1, 14, 2, 64, 32, "f16", new=509, past=7683),
        # A document in one pass.
        "prompt 8192": _case("prompt", 1, 32, 8, 128, 64, new=8192),
        # The second half of a longer one under a sliding window with the first four tokens in sight.
        "window 1024 of 16k": _case("prompt", 1, 16, 4, 128, 128, new=8192, past=8191, window=1024, sinks=4),
        # The next word for one user with a short text.
        "decode 517": _case("decode", 1, 16, 8, 128, 16, past=516),
        # A batch of users with uneven texts.
        "decode 64 x 8k": _case("decode", 64, 32, 8, 128, 64, past=8100),
        # One user with a very long text: the cache's length is all there is to split.
        "decode 131k": _case("decode", 1, 32, 4, 128, 64, "f16", past=131000),
        # A short cache past its budget, as after a few hundred words.
        "evict 1100 to 512": _case("evict", 1, 16, 8, 128, 16, past=1099, budget=512, sinks=4, recent=128),
        # A batch of long ones.
        "evict 8 x 16k to 4k": _case("evict", 8, 32, 8, 128, 64, past=16383, budget=4096, sinks=4, recent=1000),
    }
    return [dict(case, name=name) for name, case in named.items()]


def draw(rng):
    most = [max(_size(c)[i] for c in listed()) for i in range(2)]
    while True:
        case = _draw_one(rng)
        if all(n <= m for n, m in zip(_size(case), most)):
            return case


def _size(case):
    """What a pass of the plain form holds (scores, or the cache), and what the call has to move, as a bound on drawn cases."""
    lens, new = _lens(case)
    held = case["batch"] * case["kv_heads"] * max(lens) * case["head_dim"]
    if case["kind"] == "prompt":
        held = max(held, case["batch"] * case["q_heads"] * max(new) * max(lens))
    return held, work(case)["bytes"] + work(case)["flops"] / 200.0


def _draw_one(rng):
    def log_int(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    kind = rng.choice(["append", "prompt", "prompt", "decode", "decode", "evict"])
    kv_heads, group = rng.choice([1, 2, 4, 5, 8]), rng.choice([1, 2, 4, 4, 5, 7, 8, 16])
    head_dim, dtype, page = rng.choice([64, 128, 128]), rng.choice(["bf16", "bf16", "f16"]), rng.choice([16, 32, 64, 128])
    batch = rng.choice([1, 1, 2, 3, log_int(4, 100)])
    case = _case(kind, batch, kv_heads * group, kv_heads, head_dim, page, dtype, ragged=rng.random() < 0.8, empty=batch > 1 and rng.random() < 0.25)
    if kind == "append":
        case["new"], case["past"] = rng.choice([1, log_int(2, 8000)]), rng.choice([0, log_int(1, 4000)])
        case["rot"], case["interleaved"] = rng.choice([0, 0, head_dim // 2]), rng.random() < 0.3
        case["shift"] = rng.choice([0, log_int(1, 3000)])
    elif kind == "evict":
        case["past"] = log_int(40, 33000)
        case["budget"] = max(8, int(case["past"] * rng.uniform(0.2, 1.1)))
        case["sinks"], case["recent"] = rng.choice([0, 1, 4]), int(case["budget"] * rng.uniform(0, 0.5))
    else:
        case["new"] = log_int(2, 8192) if kind == "prompt" else 1
        case["past"] = rng.choice([0, log_int(1, 16000)]) if kind == "prompt" else log_int(1, 131000)
        if rng.random() < 0.4:
            case["window"], case["sinks"] = log_int(16, 4096), rng.choice([0, 1, 4, 130])
    return case


# ---------------------------------------------------------------------------------------------------- sizes

def _lens(case):
    """(slots filled after the call, tokens of the call) for each sequence."""
    lens, new = [], []
    for i in range(case["batch"]):
        share = 0.15 + 0.85 * ((1.0 + i * 0.6180339887) % 1.0) if case["ragged"] and i else 1.0
        n, p = max(1, round(case["new"] * share)), round(case["past"] * share)
        if case["empty"] and i == case["batch"] - 1:
            n = p = 0
        new.append(n)
        lens.append(n + p)
    if case["kind"] in ("decode", "evict"):
        new = [1] * case["batch"]
    return lens, new


def _pages(n, page):
    return (n + page - 1) // page


def _pairs(case, end, n):
    """(query, key) pairs in sight for the last n of `end` tokens."""
    w, s = case["window"], case["sinks"]
    total = 0
    for p in range(end - n, end):
        total += p + 1 if w == 0 else min(w, p + 1) + min(s, max(0, p + 1 - w))
    return total


def _keys(case, end, n):
    """Slots that some of the last n of `end` tokens see."""
    w, s = case["window"], case["sinks"]
    if end == 0:
        return 0
    first = 0 if w == 0 else max(0, end - n - w + 1)
    return end - first + min(s, first)


def work(case):
    lens, new = _lens(case)
    d, hq, hk = case["head_dim"], case["q_heads"], case["kv_heads"]
    tokens = sum(new)
    if case["kind"] == "append":
        rot = case["rot"] or d
        return {"bytes": 2 * tokens * d * (hq + 2 * hk) * 2 + 4 * tokens * rot, "flops": 10 * tokens * d * (hq + hk)}
    if case["kind"] == "prompt":
        pairs = sum(_pairs(case, end, n) for end, n in zip(lens, new))
        keys = sum(_keys(case, end, n) for end, n in zip(lens, new))
        return {"bytes": 2 * tokens * hq * d * 2 + 4 * tokens * hq + 2 * keys * hk * d * 2, "flops": 4 * pairs * hq * d}
    if case["kind"] == "decode":
        keys = sum(_keys(case, end, 1) for end in lens)
        return {"bytes": 2 * case["batch"] * hq * d * 2 + 4 * case["batch"] * hq + 2 * keys * hk * d * 2 + 8 * sum(lens) * hk, "flops": 4 * keys * hq * d}
    kept = sum(min(n, case["budget"]) for n in lens)
    return {"bytes": 4 * sum(lens) * hk + 2 * 2 * kept * hk * d * 2 + 2 * 4 * kept * hk, "flops": 0}


# ---------------------------------------------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    host = torch.Generator()
    host.manual_seed(seed)
    dtype, d, hq, hk, page, batch = DTYPES[case["dtype"]], case["head_dim"], case["q_heads"], case["kv_heads"], case["page"], case["batch"]
    lens, new = _lens(case)

    def normal(*shape, std=1.0):
        return (std * torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)).to(dtype)

    per_seq = [_pages(n, page) for n in lens]
    kept_pages = _pages(case["budget"], page) if case["kind"] == "evict" else 0
    pages = sum(per_seq) + batch * kept_pages + 3
    width = max(1, max(per_seq))
    order = torch.randperm(pages, generator=host).to(torch.int32)  # a pool that has been in use for a while
    table, at = torch.full((batch, width), -1, dtype=torch.int32), 0
    for i, n in enumerate(per_seq):
        table[i, :n] = order[at:at + n]
        at += n
    s = {"case": case, "k": normal(pages, hk, page, d), "v": normal(pages, hk, page, d), "table": table.cuda(),
         "lens": torch.tensor(lens, dtype=torch.int32).cuda(), "scale": 1.0 / math.sqrt(d)}
    tokens = sum(new)
    s["cu"] = torch.tensor([0] + new, dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()
    if case["kind"] == "append":
        s["qkv"] = normal(tokens, (hq + 2 * hk) * d, std=2.0)
        s["q_norm"], s["k_norm"] = 1.0 + normal(d, std=0.1), 1.0 + normal(d, std=0.1)
        rot, rows = case["rot"] or d, max(lens) + case["shift"]
        angle = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * ROPE_BASE ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
        s["rope"] = torch.cat([angle.sin(), angle.cos()], 1).float()
        position = [end - n + i + case["shift"] for end, n in zip(lens, new) for i in range(n)]
        s["positions"] = torch.tensor(position, dtype=torch.int32).cuda()
        s["q"] = torch.empty(tokens, hq, d, dtype=dtype, device="cuda")
        return s
    # Scores with a deviation of 1.5: a few keys stand out for each query.
    s["q"], s["max_new"] = normal(tokens, hq, d, std=1.5), max(new)
    if case["kind"] in ("decode", "evict"):
        # What the tokens have got so far: a few heavy hitters, many that got next to nothing, equal values among them.
        heavy = torch.randn((batch, hk, width * page), generator=g, device="cuda", dtype=torch.float32)
        s["weights"] = torch.where(heavy < -1.0, 0.0, torch.exp(2.0 * heavy))
        s["weights_out"] = torch.zeros_like(s["weights"])
    if case["kind"] == "evict":
        s["table_out"] = order[at:at + batch * kept_pages].reshape(batch, kept_pages).cuda()
        s["weights_out"] = torch.zeros((batch, hk, kept_pages * page), device="cuda")
    return s


# ---------------------------------------------------------------------------------------------------- one pass

def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    from owoinfer_b200 import ops
    case = s["case"]
    cache = ops.PagedCache(s["k"], s["v"], s["table"], s["lens"])
    if case["kind"] == "append":
        ops.qk_norm_rope_append(s["qkv"], cache, s["cu"], s["q_norm"], s["k_norm"], s["rope"], positions=s["positions"], eps=EPS,
                                interleaved=case["interleaved"], out=s["q"])
        return {"q": s["q"], "k": s["k"], "v": s["v"]}
    if case["kind"] == "prompt":
        out, lse = ops.attention_paged(s["q"], cache, s["cu"], s["max_new"], s["scale"], window=case["window"], sinks=case["sinks"])
        return {"out": out, "lse": lse}
    if case["kind"] == "decode":
        out, lse = ops.attention_paged_decode(s["q"], cache, s["scale"], window=case["window"], sinks=case["sinks"],
                                              weights=s["weights"], weights_out=s["weights_out"])
        return {"out": out, "lse": lse, "weights": s["weights_out"]}
    kept, lens = ops.kv_evict(cache, s["weights"], s["table_out"], case["budget"], sinks=case["sinks"], recent=case["recent"],
                              weights_out=s["weights_out"])
    return {"kept": kept, "lens": lens, "weights": s["weights_out"], "k": s["k"], "v": s["v"]}


def _gather(pool, table):
    """[batch, kv_heads, slots, head_dim] of the pages of `table` in 32 bits (a page that is not there reads as some other)."""
    x = pool[table.clamp(min=0).long()].permute(0, 2, 1, 3, 4)
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[4]).float()


def _rotated_norm(x, weight, sin, cos, interleaved):
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()
    half = sin.shape[-1]
    sin, cos = sin[:, None], cos[:, None]
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, rest], -1)


def _tokens(s, n):
    """For each of n tokens: its sequence, its place among the call's tokens of that sequence, its slot in the cache."""
    cu = s["cu"].long()
    token = torch.arange(n, device=cu.device)
    seq = torch.searchsorted(cu[1:], token, right=True)
    place = token - cu[seq]
    return seq, place, s["lens"].long()[seq] - (cu[seq + 1] - cu[seq]) + place


def _softmax(scores, seen):
    """Weights and the logarithm of their sum over the last axis; a row that sees nothing has zeros and -inf."""
    scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    scores.sub_(top).exp_()
    total = scores.sum(-1, keepdim=True)
    scores.div_(torch.where(total == 0.0, 1.0, total))
    return scores, (top + total.log())[..., 0]


def _seen(case, slot, keys):
    """Whether the query at `slot` sees each key slot."""
    key = torch.arange(keys, device=slot.device)
    seen = key <= slot[..., None]
    if case["window"]:
        seen &= (key < case["sinks"]) | (slot[..., None] - key < case["window"])
    return seen


def _run_plain(s):
    case, dtype = s["case"], DTYPES[s["case"]["dtype"]]
    hq, hk, d, page = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
    if case["kind"] == "append":
        qkv = s["qkv"].view(-1, hq + 2 * hk, d).float()
        sin, cos = s["rope"][s["positions"].long()].chunk(2, -1)
        q = _rotated_norm(qkv[:, :hq], s["q_norm"], sin, cos, case["interleaved"])
        k = _rotated_norm(qkv[:, hq:hq + hk], s["k_norm"], sin, cos, case["interleaved"])
        seq, _, slot = _tokens(s, qkv.shape[0])
        where = s["table"].long()[seq, slot // page]
        s["k"][where, :, slot % page] = k.to(dtype)
        s["v"][where, :, slot % page] = s["qkv"].view(-1, hq + 2 * hk, d)[:, hq + hk:]
        s["q"].copy_(q)
        return {"q": s["q"], "k": s["k"], "v": s["v"]}
    if case["kind"] == "evict":
        return _evict_plain(s)
    batch, n = case["batch"], s["max_new"]
    seq, place, slot = _tokens(s, s["q"].shape[0])
    slots = torch.full((batch, n), -1, dtype=torch.int64, device="cuda")
    slots[seq, place] = slot
    q = torch.zeros((batch, n, hq, d), device="cuda")
    q[seq, place] = s["q"].float()
    k, v = _gather(s["k"], s["table"]), _gather(s["v"], s["table"])
    seen = _seen(case, slots, k.shape[2])[:, None, None]
    q = q.view(batch, n, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(batch, hk, -1, d)
    scores = (q @ k.transpose(-1, -2)).mul_(s["scale"]).view(batch, hk, hq // hk, n, -1)
    p, lse = _softmax(scores, seen)
    out = (p.view(batch, hk, -1, k.shape[2]) @ v).view(batch, hk, hq // hk, n, d).permute(0, 3, 1, 2, 4).reshape(batch, n, hq, d)
    lse = lse.permute(0, 3, 1, 2).reshape(batch, n, hq)
    got = {"out": out[seq, place].to(dtype), "lse": lse[seq, place]}
    if case["kind"] == "decode":
        # The newest token's own slot starts at what it gets in this call.
        key, last = torch.arange(k.shape[2], device="cuda"), s["lens"].long()[:, None, None] - 1
        before = torch.where(key == last, 0.0, s["weights"])
        s["weights_out"].copy_(torch.where(key <= last, before + p.sum((2, 3)), s["weights_out"]))
        got["weights"] = s["weights_out"]
    return got


def _evict_plain(s):
    case, page = s["case"], s["case"]["page"]
    budget, sinks, recent = case["budget"], case["sinks"], case["recent"]
    lens, (batch, hk, slots) = s["lens"].long()[:, None, None], s["weights"].shape
    slot = torch.arange(slots, device="cuda")
    # First tokens and last ones ahead of all others, what is not there behind them; equal weights by their slots.
    rank = torch.where((slot < sinks) | (slot >= lens - recent) | (lens <= budget), math.inf, s["weights"])
    rank = torch.where(slot >= lens, -math.inf, rank)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :budget]
    room = torch.arange(budget, device="cuda")
    count = lens.clamp(max=budget)
    kept = torch.where(room[:order.shape[-1]] < count, order, slots).sort(-1).values
    kept = torch.cat([kept, kept.new_full((batch, hk, budget - kept.shape[-1]), slots)], -1)
    there = room < count
    b, h, i = (x.expand(batch, hk, budget) for x in (torch.arange(batch, device="cuda")[:, None, None], torch.arange(hk, device="cuda")[:, None], room))
    source = torch.where(there, kept, 0)
    page_from = s["table"].long()[b, source // page].clamp(min=0)
    page_to = s["table_out"].long()[b, i // page]
    mask = there[..., None]
    for pool in (s["k"], s["v"]):
        pool[page_to, h, i % page] = torch.where(mask, pool[page_from, h, source % page], pool[page_to, h, i % page])
    weights = torch.gather(s["weights"], 2, source)
    s["weights_out"][..., :budget] = torch.where(there, weights, s["weights_out"][..., :budget])
    return {"kept": torch.where(there, kept, -1).int(), "lens": count[:, 0, 0].int(), "weights": s["weights_out"], "k": s["k"], "v": s["v"]}


# ---------------------------------------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "prompt": _exact_attention, "decode": _exact_attention, "evict": _exact_evict}[case["kind"]](case, s)


def _slots_of(case, s, i, count):
    """Page and row of the first `count` slots of sequence i."""
    at = torch.arange(count, device="cuda")
    return s["table"][i].long()[at // case["page"]], at % case["page"]


def _exact_append(case, s):
    lens, new = _lens(case)
    hq, hk, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    rot = case["rot"] or d
    x = s["qkv"].double().reshape(-1, hq + 2 * hk, d)
    y = x[:, :hq + hk]
    y = y / (y.pow(2).sum(-1, keepdim=True) / d + EPS).sqrt()
    y[:, :hq] *= s["q_norm"].double()
    y[:, hq:] *= s["k_norm"].double()
    first = torch.arange(0, rot, 2, device="cuda") if case["interleaved"] else torch.arange(rot // 2, device="cuda")
    second = first + (1 if case["interleaved"] else rot // 2)
    sin, cos = (t[:, None] for t in s["rope"][s["positions"].long()].double().split(rot // 2, -1))
    z = y.clone()
    z[..., first] = y[..., first] * cos - y[..., second] * sin
    z[..., second] = y[..., second] * cos + y[..., first] * sin
    k, v, at = s["k"].double(), s["v"].double(), 0
    for i, (end, n) in enumerate(zip(lens, new)):
        if n:
            page, row = (t[end - n:] for t in _slots_of(case, s, i, end))
            k[page, :, row], v[page, :, row] = z[at:at + n, hq:], x[at:at + n, hq + hk:]
        at += n
    return {"q": z[:, :hq], "k": k, "v": v}


def _exact_attention(case, s):
    lens, new = _lens(case)
    hq, hk, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    weights = s["weights_out"].double() if case["kind"] == "decode" else None
    at = 0
    for i, (end, n) in enumerate(zip(lens, new)):
        rows = slice(at, at + n)
        at += n
        if end == 0 or n == 0:
            continue
        page, row = _slots_of(case, s, i, end)
        query, key = torch.arange(end - n, end, device="cuda")[:, None], torch.arange(end, device="cuda")[None]
        hidden = key > query
        if case["window"]:
            hidden |= (key >= case["sinks"]) & (query - key >= case["window"])
        for h in range(hq):
            group = h // (hq // hk)
            kh, vh = s["k"][page, group, row].double(), s["v"][page, group, row].double()
            dot = (s["q"][rows, h].double() @ kh.T) * (d ** -0.5)
            dot[hidden] = -math.inf
            lse[rows, h] = torch.logsumexp(dot, -1)
            p = (dot - lse[rows, h][:, None]).exp()
            out[rows, h] = p @ vh
            if weights is not None:
                if h % (hq // hk) == 0:
                    weights[i, group, :end - 1], weights[i, group, end - 1] = s["weights"][i, group, :end - 1].double(), 0.0
                weights[i, group, :end] += p[0]
    got = {"out": out, "lse": lse}
    return got if weights is None else dict(got, weights=weights)


def _exact_evict(case, s):
    lens, _ = _lens(case)
    page, budget = case["page"], case["budget"]
    k, v, weights = s["k"].double(), s["v"].double(), s["weights_out"].double()
    given = s["weights"].cpu().numpy()
    for i, end in enumerate(lens):
        source_page, source_row = _slots_of(case, s, i, end)
        for h in range(case["kv_heads"]):
            middle = [] if end <= budget else range(case["sinks"], end - case["recent"])
            leaving = sorted(middle, key=lambda j: (-float(given[i, h, j]), j))[budget - case["sinks"] - case["recent"]:]
            stays = torch.ones(end, dtype=torch.bool)
            stays[leaving] = False
            kept = stays.nonzero()[:, 0].cuda()
            to = torch.arange(kept.shape[0], device="cuda")
            where = s["table_out"][i].long()[to // page], h, to % page
            k[where], v[where] = k[source_page[kept], h, source_row[kept]], v[source_page[kept], h, source_row[kept]]
            weights[i, h, to] = s["weights"][i, h, kept].double()
    # (The places and lengths that are kept are whole numbers.)
    return {"kept": None, "lens": None, "weights": weights, "k": k, "v": v}
