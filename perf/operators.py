"""Performance cases of the operators around a paged key-value cache, and what they compute in plain form.

A case is a dict of plain values; its ``kind`` names the operator:

``attention``  ``ops.paged_attention``: queries of ragged sequences (one new token each, a prompt, or a part of one behind what the
               cache already holds) over keys and values in pages, with a cap on the scores, a bias by distance, a window, a prefix
``append``     ``ops.paged_rope_append``: rotary positions for q and k, k and v stored in the pages
``logprobs``   ``ops.token_logprobs``: log probability of given tokens, entropy of the distribution, the likeliest alternatives

``own`` False: :func:`run` computes the plain form, elementary torch operations in 32 bits, rounded once; True: it calls the
operators.  Sequence lengths go by the case alone (evenly spaced in their logarithm), their order and the order of the pages by the seed.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    def attention(name, **kw):
        base = dict(name=name, kind="attention", dtype="fp16", dim=128, page=16, causal=True, cap=0.0, window=0, prefix=0, slopes=False)
        return {**base, **kw}

    return [
        # one sequence of the 7B shape (32 heads, each with keys of its own) at the context of the decode benchmark: latency counts
        attention("decode_b1", heads=32, kv_heads=32, batch=1, new_lo=1, new_hi=1, past_lo=2011, past_hi=2011),
        # a served batch, every sequence at another length, four query heads to a key head
        attention("decode_b64_ragged", heads=32, kv_heads=8, batch=64, new_lo=1, new_hi=1, past_lo=37, past_hi=2047, page=32),
        # one sequence with a very long context
        attention("decode_b1_long", heads=32, kv_heads=8, batch=1, new_lo=1, new_hi=1, past_lo=131000, past_hi=131000, page=64),
        # capped scores, a window behind four tokens that always stay visible, five query heads to a key head, narrow heads
        attention("decode_b33_window", heads=40, kv_heads=8, batch=33, new_lo=1, new_hi=1, past_lo=333, past_hi=8190, dtype="bf16", dim=64,
                  cap=30.0, window=1000, prefix=4),
        # a prompt of 2048 tokens of the 7B shape, as in the benchmark
        attention("prompt_2048", heads=32, kv_heads=32, batch=1, new_lo=2048, new_hi=2048, past_lo=0, past_hi=0),
        # prompts of very different lengths in one call, bias by distance
        attention("prompts_ragged", heads=32, kv_heads=8, batch=13, new_lo=1, new_hi=1777, past_lo=0, past_hi=0, page=32, slopes=True),
        # a chunk of a long document behind what is cached already, capped scores
        attention("chunk_512_on_30000", heads=28, kv_heads=4, batch=1, new_lo=512, new_hi=512, past_lo=30000, past_hi=30000, page=64, dtype="bf16",
                  cap=50.0),
        # a long prompt
        attention("prompt_8192", heads=32, kv_heads=8, batch=1, new_lo=8192, new_hi=8192, past_lo=0, past_hi=0, page=128),
        # the new tokens of a served batch
        dict(name="append_b64", kind="append", dtype="fp16", heads=32, kv_heads=8, dim=128, rotary=128, interleaved=False, page=32, batch=64,
             new_lo=1, new_hi=1, past_lo=37, past_hi=2047),
        # prompts, half of a head rotated, neighbouring values paired
        dict(name="append_prompts", kind="append", dtype="bf16", heads=32, kv_heads=8, dim=128, rotary=64, interleaved=True, page=16, batch=5,
             new_lo=333, new_hi=4096, past_lo=0, past_hi=0),
        # what was sampled for one sequence, with five alternatives
        dict(name="logprobs_b1", kind="logprobs", dtype="fp16", rows=1, vocab=32000, top=5, banned=0.0),
        # every token of a prompt, a tenth of the vocabulary excluded
        dict(name="logprobs_prompt", kind="logprobs", dtype="fp16", rows=2048, vocab=32000, top=20, banned=0.1),
    ]


# ---------------------------------------------------------------------------------------------- more of the same ranges
def _log(rng, lo, hi):
    """Spread over the logarithm of lo..hi, odd values among them."""
    return int(min(hi, max(lo, round(lo * (hi / lo) ** rng.random()))))


HEADS = ((32, 32), (32, 8), (40, 8), (16, 2), (12, 4), (28, 4), (8, 1), (20, 20), (64, 8))


def _draw_attention(rng):
    heads, kv = rng.choice(HEADS)
    case = dict(kind="attention", dtype=rng.choice(("fp16", "fp16", "bf16")), heads=heads, kv_heads=kv, dim=rng.choice((128, 128, 64)),
                page=rng.choice((16, 32, 64, 128)), causal=True, cap=rng.choice((0.0, 0.0, 30.0, 50.0)), window=0, prefix=0,
                slopes=rng.random() < 0.2)
    what = rng.random()
    if what < 0.45:                      # one new token each
        batch = _log(rng, 1, 64)
        hi = _log(rng, 16, min(131000, 131000 * 8 // (kv * batch) + 16))
        case.update(batch=batch, new_lo=1, new_hi=1, past_lo=max(1, int(hi * rng.uniform(0.02, 1.0))), past_hi=hi)
    elif what < 0.6:                     # a few tokens each, behind a context
        batch = _log(rng, 1, 32)
        hi = _log(rng, 64, min(32768, 131000 * 8 // (kv * batch)))
        new = rng.randint(2, 16)
        case.update(batch=batch, new_lo=rng.randint(1, new), new_hi=new, past_lo=max(1, int(hi * rng.uniform(0.1, 1.0))), past_hi=hi)
    else:                                # prompts, sometimes behind a context
        batch = _log(rng, 1, 16)
        hi = _log(rng, 33, 8192 // batch)
        past = 0 if rng.random() < 0.6 else _log(rng, 16, max(16, 8192 * 2048 // (hi * batch)))
        case.update(batch=batch, new_lo=max(1, int(hi * rng.uniform(0.05, 1.0))), new_hi=hi, past_lo=past // 2, past_hi=past)
        if rng.random() < 0.1:
            case["causal"] = False
    if case["causal"] and rng.random() < 0.3:
        case["window"] = _log(rng, 16, 4096)
    if case["causal"] and rng.random() < 0.2:
        case["prefix"] = _log(rng, 1, 300)
    return case


def draw(rng):
    kind = rng.choice(("attention", "attention", "attention", "append", "logprobs"))
    if kind == "attention":
        return _draw_attention(rng)
    dtype = rng.choice(("fp16", "bf16"))
    if kind == "append":
        heads, kv = rng.choice(HEADS)
        dim = rng.choice((128, 64))
        case = dict(kind=kind, dtype=dtype, heads=heads, kv_heads=kv, dim=dim, rotary=rng.choice((dim, dim, dim // 2, dim // 4)),
                    interleaved=rng.random() < 0.4, page=rng.choice((16, 32, 64, 128)))
        if rng.random() < 0.5:
            hi = _log(rng, 16, 8192)
            return dict(case, batch=_log(rng, 1, 128), new_lo=1, new_hi=1, past_lo=int(hi * rng.uniform(0.02, 1.0)), past_hi=hi)
        batch = _log(rng, 1, 16)
        hi = _log(rng, 33, 8192 // batch)
        return dict(case, batch=batch, new_lo=max(1, int(hi * rng.uniform(0.05, 1.0))), new_hi=hi, past_lo=0, past_hi=_log(rng, 1, 2048))
    rows = _log(rng, 1, 2048)
    return dict(kind=kind, dtype=rng.choice(("fp16", "fp16", "bf16", "fp32")), rows=rows, vocab=_log(rng, 1000, min(152000, 2048 * 32000 // rows)),
                top=rng.choice((0, 1, 5, 20)), banned=rng.choice((0.0, 0.0, 0.1, 0.9)))


# ---------------------------------------------------------------------------------------------- sizes
def _spaced(lo, hi, n):
    """n whole numbers from lo to hi, evenly spaced in the logarithm of their successors."""
    if n == 1:
        return [hi]
    return [round((lo + 1) * ((hi + 1) / (lo + 1)) ** (i / (n - 1))) - 1 for i in range(n)]


def _lengths(case):
    """New tokens and tokens in the cache before them, of every sequence: the longest prompts lie behind the shortest contexts."""
    return _spaced(case["new_lo"], case["new_hi"], case["batch"]), _spaced(case["past_lo"], case["past_hi"], case["batch"])[::-1]


def _visible(case, new, past):
    """(pairs of a query and a visible key, keys that some query sees) of one sequence."""
    length = past + new
    if not case["causal"]:
        return new * length, length
    position = torch.arange(past, length, dtype=torch.int64)
    low = (position + 1 - case["window"]).clamp(min=0) if case["window"] else torch.zeros_like(position)
    always = torch.full_like(position, min(case["prefix"], length))
    pairs = always + (position + 1 - torch.maximum(low, always)).clamp(min=0)
    first = int(low[0])
    return int(pairs.sum()), length - max(0, first - int(always[0]))


# ---------------------------------------------------------------------------------------------- states
def _generator(seed, stream):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000 + stream)
    return g


def _randn(shape, dtype, g):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=g)


def _tables(positions, rotary):
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (
        -torch.arange(rotary // 2, dtype=torch.float64, device="cuda") * 2 / rotary)
    return torch.cos(angle).float(), torch.sin(angle).float()


def _paged(case, seed):
    """Lengths, first rows and page table of the case's sequences, in the seed's order: the pages of a pool that has been in use for
    a while, entries of the table that no token has reached yet hold -1."""
    g = _generator(seed, 1)
    new, past = (torch.tensor(v, dtype=torch.int64) for v in _lengths(case))
    order = torch.randperm(case["batch"], generator=torch.Generator().manual_seed(seed))
    new, length = new[order], (new + past)[order]
    used = (length + case["page"] - 1) // case["page"]
    width = int(used.max()) + 1
    pool = int(used.sum()) + 3
    table = torch.full((case["batch"], width), -1, dtype=torch.int32, device="cuda")
    place = torch.arange(width, device="cuda")[None, :] < used.cuda()[:, None]
    table[place] = torch.randperm(pool, device="cuda", generator=g)[: int(used.sum())].int()
    starts = torch.zeros(case["batch"] + 1, dtype=torch.int32)
    starts[1:] = new.cumsum(0)
    shape = (pool, case["kv_heads"], case["page"], case["dim"])
    dtype = DTYPES[case["dtype"]]
    state = dict(kind=case["kind"], k=_randn(shape, dtype, g), v=_randn(shape, dtype, g), table=table, lengths=length.int().cuda(),
                 max_query=int(new.max()), starts=None if case["new_hi"] == 1 else starts.cuda())
    return state, int(new.sum()), g


def _prepare_attention(case, seed):
    state, tokens, g = _paged(case, seed)
    state["q"] = _randn((tokens, case["heads"], case["dim"]), DTYPES[case["dtype"]], g)
    state.update(causal=case["causal"], cap=case["cap"], window=case["window"], slopes=None, prefix=None)
    if case["slopes"]:
        state["slopes"] = 2.0 ** (-8.0 * torch.arange(1, case["heads"] + 1, device="cuda", dtype=torch.float32) / case["heads"])
    if case["prefix"]:
        state["prefix"] = torch.full((case["batch"],), case["prefix"], dtype=torch.int32, device="cuda")
    return state


def _prepare_append(case, seed):
    state, tokens, g = _paged(case, seed)
    state["qkv"] = _randn((tokens, (case["heads"] + 2 * case["kv_heads"]) * case["dim"]), DTYPES[case["dtype"]], g)
    state["cos"], state["sin"] = _tables(case["new_hi"] + case["past_hi"] + 1, case["rotary"])
    state["interleaved"] = case["interleaved"]
    return state


def _prepare_logprobs(case, seed):
    g = _generator(seed, 1)
    logits = _randn((case["rows"], case["vocab"]), torch.float32, g) * 2.5
    if case["banned"]:
        logits.masked_fill_(torch.rand(case["vocab"], device="cuda", generator=g) < case["banned"], -math.inf)
    tokens = torch.randint(0, case["vocab"], (case["rows"],), dtype=torch.int32, device="cuda", generator=g)
    return dict(kind="logprobs", logits=logits.to(DTYPES[case["dtype"]]), tokens=tokens, top=case["top"])


def prepare(case, seed):
    return {"attention": _prepare_attention, "append": _prepare_append, "logprobs": _prepare_logprobs}[case["kind"]](case, seed)


# ---------------------------------------------------------------------------------------------- the plain forms
def _rows_of(state, tokens):
    """Sequence and place in it of every row, and its position."""
    lengths = state["lengths"].long()
    if state["starts"] is None:
        seq = torch.arange(tokens, device="cuda")
        return seq, torch.zeros_like(seq), lengths - 1
    starts = state["starts"].long()
    row = torch.arange(tokens, device="cuda")
    seq = torch.searchsorted(starts, row, right=True) - 1
    place = row - starts[seq]
    return seq, place, lengths[seq] - (starts[seq + 1] - starts[seq]) + place


def _plain_attention(s):
    q, table, lengths = s["q"], s["table"].clamp(min=0).long(), s["lengths"].long()
    tokens, heads, dim = q.shape
    kv = s["k"].shape[1]
    batch, longest = table.shape[0], s["max_query"]
    k, v = (s[c][table].float().transpose(1, 2).reshape(batch, kv, -1, dim) for c in "kv")
    seq, place, position = _rows_of(s, tokens)
    padded = torch.zeros((batch, longest, heads, dim), dtype=torch.float32, device="cuda")
    padded[seq, place] = q.float()
    where = torch.full((batch, longest), -1, dtype=torch.int64, device="cuda")
    where[seq, place] = position
    grouped = padded.view(batch, longest, kv, heads // kv, dim).permute(0, 2, 3, 1, 4).reshape(batch, kv, -1, dim)
    scores = (grouped @ k.transpose(2, 3)).mul_(dim ** -0.5).view(batch, kv, heads // kv, longest, -1)
    if s["cap"]:
        scores = scores.div_(s["cap"]).tanh_().mul_(s["cap"])
    key = torch.arange(k.shape[2], device="cuda")
    distance = where[:, :, None] - key
    if s["slopes"] is not None:
        scores -= s["slopes"].view(kv, -1, 1, 1) * distance.abs().float()[:, None, None]
    seen = key < lengths[:, None, None]
    if s["causal"]:
        near = distance >= 0
        if s["window"]:
            near &= distance < s["window"]
        if s["prefix"] is not None:
            near |= key < s["prefix"][:, None, None]
        seen = seen & near
    seen = seen & (where >= 0)[:, :, None]
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(dim=-1, keepdim=True).clamp(min=-1e30)
    weight = scores.sub_(top).exp_()
    total = weight.sum(dim=-1, keepdim=True)
    result = (weight.view(batch, kv, -1, k.shape[2]) @ v).view(batch, kv, heads // kv, longest, dim) / total.clamp(min=1e-30)
    return result.permute(0, 3, 1, 2, 4).reshape(batch, longest, heads, dim)[seq, place].to(q.dtype)


def _rotated(x, cos, sin, interleaved):
    """x [tokens, heads, dim]: the first 2 * (columns of cos) values of a head turned pair by pair."""
    half = cos.shape[1]
    cos, sin = cos[:, None], sin[:, None]
    a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if interleaved else (x[..., :half], x[..., half:2 * half])
    first, second = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((first, second), dim=-1).flatten(-2) if interleaved else torch.cat((first, second), dim=-1)
    return torch.cat((turned, x[..., 2 * half:]), dim=-1)


def _plain_append(s):
    kv, page, dim = s["k"].shape[1:]
    qkv = s["qkv"].view(s["qkv"].shape[0], -1, dim)
    heads = qkv.shape[1] - 2 * kv
    seq, _, position = _rows_of(s, qkv.shape[0])
    cos, sin = s["cos"][position], s["sin"][position]
    turned = _rotated(qkv[:, :heads + kv].float(), cos, sin, s["interleaved"]).to(qkv.dtype)
    where = s["table"][seq, position // page].long()
    s["k"][where, :, position % page] = turned[:, heads:]
    s["v"][where, :, position % page] = qkv[:, heads + kv:]
    return {"q": turned[:, :heads].contiguous(), "k": s["k"], "v": s["v"]}


def _plain_logprobs(s):
    x = s["logits"].float()
    x = x - x.amax(dim=-1, keepdim=True)
    log = x - x.exp().sum(dim=-1, keepdim=True).log()
    result = {"logprob": log.gather(1, s["tokens"].long()[:, None])[:, 0],
              "entropy": -torch.where(log > -math.inf, log.exp() * log, 0.0).sum(dim=-1)}
    if s["top"]:
        best = torch.sort(s["logits"], dim=-1, descending=True, stable=True).indices[:, :s["top"]]
        result.update(top_logprob=log.gather(1, best), top_token=best.int())
    return result


def run(state):
    s = state
    if not own:
        return {"attention": _plain_attention, "append": _plain_append, "logprobs": _plain_logprobs}[s["kind"]](s)
    from relax_b200 import ops

    if s["kind"] == "attention":
        return ops.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"], starts=s["starts"], max_query=s["max_query"],
                                   causal=s["causal"], window=s["window"], cap=s["cap"], slopes=s["slopes"], prefix=s["prefix"])
    if s["kind"] == "append":
        q = ops.paged_rope_append(s["qkv"], s["cos"], s["sin"], s["k"], s["v"], s["table"], s["lengths"], starts=s["starts"],
                                  interleaved=s["interleaved"])
        return {"q": q, "k": s["k"], "v": s["v"]}
    r = ops.token_logprobs(s["logits"], s["tokens"], top=s["top"])
    result = {"logprob": r.logprob, "entropy": r.entropy}
    if s["top"]:
        result.update(top_logprob=r.top_logprob, top_token=r.top_token)
    return result


# ---------------------------------------------------------------------------------------------- what a pass must do
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * (12 + 8 * case["top"]), "flops": 6 * n}
    new, past = _lengths(case)
    tokens = sum(new)
    pages = sum(-(-(a + b) // case["page"]) for a, b in zip(new, past))
    around = 4 * (pages + 2 * case["batch"])
    if case["kind"] == "append":
        row = (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
        turned = (case["heads"] + case["kv_heads"]) * case["rotary"]
        return {"bytes": tokens * (2 * row * size + 4 * case["rotary"]) + around, "flops": 3 * tokens * turned}
    counts = [_visible(case, a, b) for a, b in zip(new, past)]
    pairs, keys = sum(c[0] for c in counts), sum(c[1] for c in counts)
    return {"bytes": 2 * size * case["dim"] * (tokens * case["heads"] + keys * case["kv_heads"]) + around,
            "flops": 4 * case["dim"] * case["heads"] * pairs}


# ---------------------------------------------------------------------------------------------- the same in 64 bits
def _exact_attention(case, s):
    """Sequence by sequence and head by head, from the definition."""
    heads, group, page = case["heads"], case["heads"] // case["kv_heads"], case["page"]
    result = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lengths = s["lengths"].tolist()
    starts = s["starts"].tolist() if s["starts"] is not None else list(range(case["batch"] + 1))
    for b, length in enumerate(lengths):
        pages = s["table"][b, : -(-length // page)].long()
        rows = slice(starts[b], starts[b + 1])
        i = torch.arange(length - (starts[b + 1] - starts[b]), length, device="cuda", dtype=torch.float64)[:, None]
        j = torch.arange(length, device="cuda", dtype=torch.float64)[None, :]
        if case["causal"]:
            hidden = i < j
            if case["window"]:
                hidden = hidden | (i - j > case["window"] - 1)
            hidden = hidden & (j > case["prefix"] - 1)
        for h in range(heads):
            keys, values = (s[c][pages, h // group].double().reshape(-1, case["dim"])[:length] for c in "kv")
            x = s["q"][rows, h].double() @ keys.T / math.sqrt(case["dim"])
            if case["cap"]:
                x = case["cap"] * torch.tanh(x / case["cap"])
            if case["slopes"]:
                x = x - 2.0 ** (-8.0 * (h + 1) / heads) * (i - j).abs()
            if case["causal"]:
                x = x.masked_fill(hidden, -math.inf)
            result[rows, h] = torch.softmax(x, dim=1) @ values
    return result


def _exact_append(case, s):
    """Pair (a, b) at position t as the complex number a + ib times exp(i t w)."""
    kv, page, dim, half = case["kv_heads"], case["page"], case["dim"], case["rotary"] // 2
    cos, sin = s["cos"].double(), s["sin"].double()
    k, v = s["k"].double(), s["v"].double()
    qkv = s["qkv"].double().view(-1, case["heads"] + 2 * kv, dim)
    q = torch.empty((qkv.shape[0], case["heads"], dim), dtype=torch.float64, device="cuda")
    starts = s["starts"].tolist() if s["starts"] is not None else list(range(case["batch"] + 1))
    for b, length in enumerate(s["lengths"].tolist()):
        new = starts[b + 1] - starts[b]
        at = torch.arange(length - new, length, device="cuda")
        x = qkv[starts[b]:starts[b + 1]].clone()
        part = x[:, : case["heads"] + kv, : 2 * half]
        pairs = part.unflatten(-1, (half, 2)) if case["interleaved"] else part.unflatten(-1, (2, half)).transpose(-1, -2)
        turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * torch.complex(cos[at], sin[at])[:, None])
        part.copy_(turned.flatten(-2) if case["interleaved"] else turned.transpose(-1, -2).flatten(-2))
        q[starts[b]:starts[b + 1]] = x[:, : case["heads"]]
        pages = s["table"][b].long()[at // page]
        k[pages, :, at % page] = x[:, case["heads"]:case["heads"] + kv]
        v[pages, :, at % page] = x[:, case["heads"] + kv:]
    return {"q": q, "k": k, "v": v}


def _exact_logprobs(case, s):
    x = s["logits"].double()
    total = torch.logsumexp(x, dim=1)
    rows = torch.arange(case["rows"], device="cuda")
    p = torch.exp(x - total[:, None])
    result = {"logprob": x[rows, s["tokens"].long()] - total, "entropy": total - torch.where(p > 0, p * x, 0.0).sum(dim=1)}
    if case["top"]:
        # by value, equal ones by index
        order = torch.argsort(s["logits"].float(), dim=1, descending=True, stable=True)[:, : case["top"]]
        result.update(top_logprob=torch.gather(x, 1, order) - total[:, None], top_token=order.int())
    return result


def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "append": _exact_append, "logprobs": _exact_logprobs}[case["kind"]](case, s)
