"""The calls around a text decoder's attention: what goes into its INT8 or FP8 projections, what is added beside them, what is read off its logits.

The language model in front of the image model serves several users at once, each perhaps with an adapter of his own. The kinds:

  norm      ops.add_rms_norm_quantize: the residual stream takes up a layer's output; its root-mean-square norm leaves in 8 bits, with a
            scale for each token or each group of channels, for the projection that follows
  lora      ops.lora_add: beside a projection that all tokens share, the low-rank adapter of each token's request
  logprobs  ops.token_logprobs: the log probability and rank of given tokens, the entropy, and the most probable alternatives

The plain forms below are elementary operations in 32 bits, rounded once. Codes of 8-bit integers are returned as the values that they stand
for, in 16 bits (a value on the border between two codes may go either way); those of e4m3 as they are, beside their scales.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6
LARGEST = {"int8": 127.0, "e4m3": 448.0}
SMALLEST_SCALE = 1e-30


def _norm(tokens, dim, dtype="bf16", stream="f32", kind="int8", group=0, both=False):
    """stream: type of the residual stream; group: channels to a scale (0: all of a token's); both: the norm in 16 bits besides."""
    return {"kind": "norm", "tokens": tokens, "dim": dim, "dtype": dtype, "stream": stream, "codes": kind, "group": group, "both": both}


def _lora(tokens, dim, width, rank, adapters, sequences, dtype="bf16", uneven=False, some=False):
    """dim, width: of the projection's input and output; sequences: requests that the tokens belong to; uneven: adapters have ranks below
    `rank` too; some: every fourth request has no adapter."""
    return {"kind": "lora", "tokens": tokens, "dim": dim, "width": width, "rank": rank, "adapters": adapters, "sequences": sequences, "dtype": dtype,
            "uneven": uneven, "some": some}


def _logprobs(rows, vocab, top, dtype="bf16", masked=False, padded=0, heat=1.0):
    """masked: most tokens are not allowed (minus infinity), as where a grammar says what may follow; padded: columns of the logits behind
    the vocabulary; heat: the temperature that the logits are divided by."""
    return {"kind": "logprobs", "rows": rows, "vocab": vocab, "top": top, "dtype": dtype, "masked": masked, "padded": padded, "heat": heat}


def listed():
    named = {
        # One user, one token: twice a layer between two words. Latency alone.
        "norm one token": _norm(1, 2048),
        # A batch of users with a token each, ahead of an FP8 projection with a scale for every 128 channels.
        "norm 96 tokens": _norm(96, 5120, stream="bf16", kind="e4m3", group=128),
        # Prompts of uneven lengths in one pass, some with adapters, which read the norm in 16 bits.
        "norm 2011 tokens": _norm(2011, 4096, both=True),
        # A long document through a wide layer.
        "norm 16k tokens": _norm(16384, 8192, stream="bf16", kind="e4m3"),
        # One user with an adapter.
        "lora one token": _lora(1, 2048, 2048, 16, 4, 1),
        # A batch of users, a token each, most with an adapter of their own, beside a fused projection to queries, keys and values.
        "lora 64 users": _lora(64, 4096, 6144, 16, 48, 64, uneven=True, some=True),
        # A few short prompts, half precision, beside a feed-forward layer's projection.
        "lora 517 tokens": _lora(517, 2048, 11008, 32, 3, 5, "f16"),
        # Long prompts.
        "lora 8k tokens": _lora(8191, 4096, 4096, 64, 6, 7, some=True),
        # The next word of one user, with the alternatives that an interface shows.
        "logprobs one row": _logprobs(1, 150001, 5),
        # A batch of users, logits in 32 bits, behind a temperature.
        "logprobs 64 rows": _logprobs(64, 131072, 20, "f32", heat=0.7),
        # What a grammar allows: nearly everything is minus infinity.
        "logprobs masked": _logprobs(509, 32003, 8, "f16", masked=True, padded=61),
        # The score of a prompt under the model, token by token.
        "logprobs 4k rows": _logprobs(4096, 160000, 1),
    }
    return [dict(case, name=name) for name, case in named.items()]


def draw(rng):
    most = {}
    for c in listed():
        most[c["kind"]] = max(most.get(c["kind"], 0), work(c)["bytes"] + work(c)["flops"] / 200.0)
    while True:
        case = _draw_one(rng)
        if work(case)["bytes"] + work(case)["flops"] / 200.0 <= most[case["kind"]]:
            return case


def _draw_one(rng):
    def log_int(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    kind = rng.choice(["norm", "lora", "logprobs"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if kind == "norm":
        group = rng.choice([0, 0, 128, 64])
        dim = 128 * log_int(4, 128) if group else 16 * log_int(16, 1024)
        dtype = rng.choice([dtype, dtype, "f32"])
        return _norm(log_int(1, 16384), dim, dtype, rng.choice([dtype, "f32"]), rng.choice(["int8", "e4m3"]), group, rng.random() < 0.3)
    if kind == "lora":
        tokens = rng.choice([log_int(1, 200), log_int(1, 8191)])
        return _lora(tokens, 16 * log_int(32, 512), 16 * log_int(32, 900), rng.choice([8, 16, 16, 32, 64, 128]), log_int(1, 64), min(tokens, log_int(1, 64)), dtype,
                     rng.random() < 0.4, rng.random() < 0.4)
    return _logprobs(log_int(1, 4096), log_int(1000, 200000), rng.choice([0, 1, 5, 20, 32]), rng.choice([dtype, "f32"]), rng.random() < 0.25,
                     rng.choice([0, 0, log_int(1, 500)]), rng.choice([1.0, 1.0, rng.uniform(0.3, 2.0)]))


# ---------------------------------------------------------------------------------------------------- sizes

def _ranks(case):
    return [max(1, case["rank"] // (1 << i % 3)) if case["uneven"] else case["rank"] for i in range(case["adapters"])]


def _requests(case):
    """For each request its tokens and its adapter (-1: none). Tokens of a request follow one another."""
    r = random.Random(case["tokens"] * 1000003 + case["adapters"])
    cuts = sorted(r.sample(range(1, case["tokens"]), case["sequences"] - 1))
    counts = [b - a for a, b in zip([0] + cuts, cuts + [case["tokens"]])]
    return [(n, -1 if case["some"] and i % 4 == 3 else r.randrange(case["adapters"])) for i, n in enumerate(counts)]


def work(case):
    if case["kind"] == "norm":
        n = case["tokens"] * case["dim"]
        size = {"bf16": 2, "f16": 2, "f32": 4}
        scales = case["tokens"] * (case["dim"] // case["group"] if case["group"] else 1)
        return {"bytes": n * (size[case["dtype"]] + 2 * size[case["stream"]] + 1 + (2 if case["both"] else 0)) + 4 * scales, "flops": 8 * n}
    if case["kind"] == "lora":
        ranks, requests = _ranks(case), _requests(case)
        used = sum(ranks[a] for a in {a for _, a in requests if a >= 0})
        sides = case["dim"] + case["width"]
        return {"bytes": 2 * case["tokens"] * (case["dim"] + 2 * case["width"]) + 2 * used * sides, "flops": sum(2 * n * ranks[a] * sides for n, a in requests if a >= 0)}
    cells = case["rows"] * case["vocab"]
    return {"bytes": cells * (4 if case["dtype"] == "f32" else 2) + case["rows"] * (20 + 8 * case["top"]), "flops": 6 * cells}


# ---------------------------------------------------------------------------------------------------- inputs

def _make(case, seed):
    """The inputs as tensors on the GPU, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, to=dtype):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(std).to(to)

    s = {"case": case}
    if case["kind"] == "norm":
        # A few channels of the stream are much larger than the rest, as they are in trained models.
        loud = torch.where(torch.rand(case["dim"], generator=g, device="cuda") < 0.005, 20.0, 1.0)
        s["x"] = normal(case["tokens"], case["dim"])
        s["stream"] = (normal(case["tokens"], case["dim"], std=3.0, to=torch.float32) * loud).to(DTYPES[case["stream"]])
        s["weight"] = (1.0 + normal(case["dim"], std=0.2, to=torch.float32)).to(dtype)
    elif case["kind"] == "lora":
        dim, width, rank, n = case["dim"], case["width"], case["rank"], case["adapters"]
        s["x"], s["y"] = normal(case["tokens"], dim), normal(case["tokens"], width)
        s["a"], s["b"] = normal(n, rank, dim, std=dim ** -0.5), normal(n, width, rank, std=0.5 * rank ** -0.5)
        s["scales"] = 0.5 + torch.rand(n, generator=g, device="cuda")
        s["ranks"] = torch.tensor(_ranks(case), dtype=torch.int32).cuda() if case["uneven"] else None
        s["adapter"] = torch.tensor([a for count, a in _requests(case) for _ in range(count)], dtype=torch.int32).cuda()
    else:
        rows, vocab = case["rows"], case["vocab"]
        logits = normal(rows, vocab + case["padded"], std=2.5)
        if case["masked"]:
            hidden = torch.rand(logits.shape, generator=g, device="cuda") > 0.002
            hidden[:, rows % vocab] = False
            logits.masked_fill_(hidden, -math.inf)
        # Half of the tokens are what the model would say itself, the others any.
        any_token = torch.randint(vocab, (rows,), generator=g, device="cuda")
        s["logits"] = logits[:, :vocab]
        s["targets"] = torch.where(torch.arange(rows, device="cuda") % 2 == 0, s["logits"].argmax(-1), any_token)
    return s


def prepare(case, seed):
    s = _make(case, seed)
    if case["kind"] == "norm":
        tokens, dim = s["x"].shape
        s["stream_out"] = torch.empty_like(s["stream"])
        s["y"] = torch.empty((tokens, dim), dtype=_norm_type(case), device="cuda") if case["both"] else None
        s["values"] = torch.empty((tokens, dim), dtype=torch.bfloat16, device="cuda") if case["codes"] == "int8" else None
    elif case["kind"] == "lora":
        s["out"] = torch.empty_like(s["y"])
        if own:
            from owoinfer_b200 import ops
            s["adapters"] = ops.LoraAdapters(s["a"], s["b"], s["scales"], s["ranks"])
            s["plan"] = ops.LoraPlan(s["adapter"], case["adapters"])  # (of a step's tokens: every layer and projection uses it)
    return s


def _norm_type(case):
    return torch.bfloat16 if case["dtype"] == "f32" else DTYPES[case["dtype"]]


# ---------------------------------------------------------------------------------------------------- one pass

def run(s):
    return (_run_own if own else _run_plain)(s)


def _norm_outputs(s, q, scale):
    got = {"stream": s["stream_out"], "scale": scale}
    if s["y"] is not None:
        got["y"] = s["y"]
    if s["values"] is None:
        return dict(got, codes=q)
    dim = q.shape[1]
    by_group = (q.shape[0], scale.numel() // q.shape[0], -1)
    torch.mul(q.view(by_group), scale.view(by_group[0], by_group[1], 1), out=s["values"].view(by_group[0], by_group[1], dim // by_group[1]))
    return dict(got, values=s["values"])


def _run_own(s):
    from owoinfer_b200 import ops
    case = s["case"]
    if case["kind"] == "norm":
        q, scale = ops.add_rms_norm_quantize(s["x"], s["weight"], s["stream"], eps=EPS, dtype=torch.int8 if case["codes"] == "int8" else torch.float8_e4m3fn,
                                             group=case["group"], residual_out=s["stream_out"], norm_out=s["y"])
        return _norm_outputs(s, q, scale)
    if case["kind"] == "lora":
        return ops.lora_add(s["y"], s["x"], s["adapters"], s["plan"], out=s["out"])
    got = ops.token_logprobs(s["logits"], s["targets"], top=case["top"], scale=1.0 / case["heat"])
    return _logprob_outputs(case, got.logprobs, got.ranks, got.entropy, got.lse, got.top_logprobs, got.top_tokens)


def _logprob_outputs(case, logprobs, ranks, entropy, lse, top_logprobs, top_tokens):
    got = {"logprobs": logprobs, "ranks": ranks, "entropy": entropy, "lse": lse}
    if case["top"]:
        got |= {"top_logprobs": top_logprobs, "top_tokens": top_tokens}
    return got


def _run_plain(s):
    case = s["case"]
    if case["kind"] == "norm":
        tokens, dim = s["x"].shape
        total = s["x"].float() + s["stream"].float()
        s["stream_out"].copy_(total)
        y = total * torch.rsqrt(total.square().mean(-1, keepdim=True) + EPS) * s["weight"].float()
        if s["y"] is not None:
            s["y"].copy_(y)
        y = y.view(tokens, -1, case["group"] or dim)
        scale = (y.abs().amax(-1, keepdim=True) / LARGEST[case["codes"]]).clamp(min=SMALLEST_SCALE)
        q = (y / scale).view(tokens, dim)
        q = q.round().to(torch.int8) if case["codes"] == "int8" else q.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
        return _norm_outputs(s, q, scale.view(tokens, -1) if case["group"] else scale.view(tokens))
    if case["kind"] == "lora":
        n, rank, dim = s["a"].shape
        mine = s["adapter"][:, None] == torch.arange(n, device="cuda")
        mine = mine[:, :, None].expand(-1, -1, rank)
        if s["ranks"] is not None:
            mine = mine & (torch.arange(rank, device="cuda") < s["ranks"][:, None])
        low = (s["x"].float() @ s["a"].float().view(n * rank, dim).T).view(-1, n, rank) * s["scales"][:, None]
        low = torch.where(mine, low, 0.0).view(-1, n * rank)
        s["out"].copy_(s["y"].float() + low @ s["b"].float().transpose(1, 2).reshape(n * rank, -1))
        return s["out"]
    z = s["logits"].float() / case["heat"]
    rows = torch.arange(z.shape[0], device="cuda")
    top = z.amax(-1, keepdim=True)
    e = (z - top).exp_()
    total = e.sum(-1, keepdim=True)
    lse = (top + total.log())[:, 0]
    mean = torch.where(e == 0.0, 0.0, e * (z - top)).sum(-1, keepdim=True) / total
    entropy = (total.log() - mean)[:, 0]
    del e
    # The order goes by the logits as they came: what is divided may round two of them to one value.
    logits, mine = s["logits"], s["logits"][rows, s["targets"]][:, None]
    before = (logits > mine) | ((logits == mine) & (torch.arange(z.shape[1], device="cuda") < s["targets"][:, None]))
    ranks = (before.sum(-1) + 1).to(torch.int32)
    del before
    top_tokens = torch.sort(logits, dim=-1, descending=True, stable=True)[1][:, :case["top"]] if case["top"] > 1 else logits.argmax(-1, keepdim=True)
    return _logprob_outputs(case, z[rows, s["targets"]] - lse, ranks, entropy, lse, z.gather(-1, top_tokens) - lse[:, None], top_tokens.to(torch.int32))


# ---------------------------------------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    s = _make(case, seed)
    if case["kind"] == "norm":
        return _exact_norm(s, case)
    if case["kind"] == "lora":
        out = s["y"].double()
        ranks = _ranks(case)
        start = 0
        for count, adapter in _requests(case):
            t = slice(start, start + count)
            start += count
            if adapter >= 0:
                r = ranks[adapter]
                low = s["x"][t].double() @ s["a"][adapter, :r].double().T
                out[t] += s["scales"][adapter].double() * (low @ s["b"][adapter, :, :r].double().T)
        return out
    return _exact_logprobs(s, case)


def _exact_norm(s, case):
    parts = []
    for x, stream in zip(s["x"].split(2048), s["stream"].split(2048)):
        total = x.double() + stream.double()
        y = s["weight"].double() * total / (total.pow(2).sum(1, keepdim=True) / case["dim"] + EPS).sqrt()
        groups = y.reshape(len(y), case["dim"] // case["group"], case["group"]) if case["group"] else y[:, None]
        scale = torch.linalg.vector_norm(groups, math.inf, dim=2, keepdim=True) / LARGEST[case["codes"]]
        scale = torch.maximum(scale, torch.full_like(scale, SMALLEST_SCALE))
        if case["codes"] == "int8":
            values = {"values": (torch.round(groups / scale) * scale).reshape(y.shape)}
        else:
            values = {"codes": _e4m3(groups / scale).reshape(y.shape)}
        parts.append(dict(values, stream=total, scale=scale[..., 0] if case["group"] else scale[:, 0, 0], **({"y": y} if case["both"] else {})))
    return {k: torch.cat([p[k] for p in parts]) for k in parts[0]}


def _e4m3(v):
    """The nearest e4m3 values (three bits behind the leading one, steps of 2^-9 below 2^-6), ties to even."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(v / step) * step


def _exact_logprobs(s, case):
    parts = []
    for row, target in zip(s["logits"].split(256), s["targets"].split(256)):
        z = row.double() / case["heat"]
        p = torch.softmax(z, -1)
        lse = torch.logsumexp(z, -1)
        entropy = torch.special.entr(p).sum(-1)
        own_logit = z.gather(1, target[:, None])
        # (ranks and tokens are whole numbers: the plain form's)
        got = {"logprobs": own_logit[:, 0] - lse, "entropy": entropy, "lse": lse}
        if case["top"]:
            got["top_logprobs"] = z.topk(case["top"], -1)[0] - lse[:, None]
        parts.append(got)
    return dict({k: torch.cat([p[k] for p in parts]) for k in parts[0]}, ranks=None)
