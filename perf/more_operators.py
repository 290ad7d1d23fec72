"""Performance cases of the operators of a decode step that stays on the GPU, and what they compute in plain form.

A case is a dict of plain values; its ``kind`` names the operator:

``plan``       ``ops.paged_plan``: page table, free list, rows and slots of a call from the lengths of its sequences
``append``     ``ops.paged_rope_append`` over pages in 8 bits: rotary positions for q and k, k and v quantised with a scale for 16 tokens of a head
``attention``  ``ops.paged_attention`` over pages in 8 bits: one new token each, prompts, or a part of one behind what the cache holds
``sample``     ``ops.sample_tokens``: temperature, top-k, top-p and min-p, from a random number for each row

``own`` False: :func:`run` computes the plain form, elementary torch operations in 32 bits (sampling: 64), rounded once; True: it calls the
operators.  Sequence lengths go by the case alone (evenly spaced in their logarithm), their order and the order of the pages by the seed.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
E4M3 = torch.float8_e4m3fn
BLOCK = 16                              # tokens that share a scale
MOST = 448.0                            # the largest e4m3 value


def listed():
    def attention(name, **kw):
        base = dict(name=name, kind="attention", dtype="fp16", dim=128, page=16, causal=True, cap=0.0, window=0, prefix=0, slopes=False)
        return {**base, **kw}

    def sample(name, **kw):
        base = dict(name=name, kind="sample", dtype="fp16", temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mixed=False)
        return {**base, **kw}

    return [
        # the next token of a served batch: few sequences need a page
        dict(name="plan_b64", kind="plan", page=16, batch=64, new_lo=1, new_hi=1, past_lo=37, past_hi=2047, forget=0.0),
        # requests come in with prompts of all lengths, some of them behind what is cached, others end
        dict(name="plan_prompts", kind="plan", page=32, batch=301, new_lo=1, new_hi=1500, past_lo=0, past_hi=4000, forget=0.2),
        # the new tokens of a served batch
        dict(name="append_b64", kind="append", dtype="fp16", heads=32, kv_heads=8, dim=128, rotary=128, interleaved=False, page=32, batch=64,
             new_lo=1, new_hi=1, past_lo=37, past_hi=2047),
        # prompts, half of a head rotated, neighbouring values paired
        dict(name="append_prompts", kind="append", dtype="bf16", heads=32, kv_heads=8, dim=128, rotary=64, interleaved=True, page=16, batch=5,
             new_lo=333, new_hi=4096, past_lo=0, past_hi=0),
        # one sequence of the 7B shape (32 heads, each with keys of its own) at the context of the decode benchmark: latency counts
        attention("decode_b1", heads=32, kv_heads=32, batch=1, new_lo=1, new_hi=1, past_lo=2011, past_hi=2011),
        # a served batch, every sequence at another length, four query heads to a key head
        attention("decode_b64_ragged", heads=32, kv_heads=8, batch=64, new_lo=1, new_hi=1, past_lo=37, past_hi=2047, page=32),
        # one sequence with a very long context: what 8 bits are for
        attention("decode_b1_long", heads=32, kv_heads=8, batch=1, new_lo=1, new_hi=1, past_lo=131000, past_hi=131000, page=64),
        # a prompt of 2048 tokens of the 7B shape, as in the benchmark
        attention("prompt_2048", heads=32, kv_heads=32, batch=1, new_lo=2048, new_hi=2048, past_lo=0, past_hi=0),
        # a chunk of a long document behind what is cached already, capped scores
        attention("chunk_512_on_30000", heads=28, kv_heads=4, batch=1, new_lo=512, new_hi=512, past_lo=30000, past_hi=30000, page=64, dtype="bf16",
                  cap=50.0),
        # one sequence's next token, as chat programs draw it
        sample("sample_b1", rows=1, vocab=32000, temperature=0.8, top_k=50, top_p=0.9),
        # a served batch, every request with settings of its own, greedy ones among them
        sample("sample_b64_mixed", rows=64, vocab=152000, dtype="bf16", mixed=True),
        # many rows, cut by probability alone
        sample("sample_b512_p", rows=512, vocab=32000, dtype="fp32", top_p=0.95, min_p=0.001),
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
        hi = _log(rng, 33, 4096 // batch)
        past = 0 if rng.random() < 0.6 else _log(rng, 16, max(16, 8192 * 1500 // (hi * batch)))
        case.update(batch=batch, new_lo=max(1, int(hi * rng.uniform(0.05, 1.0))), new_hi=hi, past_lo=past // 2, past_hi=past)
        if rng.random() < 0.1:
            case["causal"] = False
    if case["causal"] and rng.random() < 0.3:
        case["window"] = _log(rng, 16, 4096)
    if case["causal"] and rng.random() < 0.2:
        case["prefix"] = _log(rng, 1, 300)
    return case


def draw(rng):
    kind = rng.choice(("attention", "attention", "attention", "append", "plan", "sample", "sample"))
    if kind == "attention":
        return _draw_attention(rng)
    if kind == "sample":
        rows = _log(rng, 1, 512)
        case = dict(kind=kind, dtype=rng.choice(("fp16", "fp16", "bf16", "fp32")), rows=rows, vocab=_log(rng, 1000, min(152000, 512 * 32000 // rows)),
                    temperature=round(rng.uniform(0.3, 1.5), 2), top_k=0, top_p=1.0, min_p=0.0, mixed=rng.random() < 0.3)
        if rng.random() < 0.5:
            case["top_k"] = _log(rng, 1, 1000)
        if rng.random() < 0.5:
            case["top_p"] = round(rng.uniform(0.1, 0.99), 3)
        if rng.random() < 0.3:
            case["min_p"] = round(rng.uniform(0.001, 0.2), 3)
        return case
    case = dict(kind=kind, page=rng.choice((16, 32, 64, 128)))
    if rng.random() < 0.5:               # one new token each
        hi = _log(rng, 16, 8192)
        case.update(batch=_log(rng, 1, 128), new_lo=1, new_hi=1, past_lo=int(hi * rng.uniform(0.02, 1.0)), past_hi=hi)
    else:
        batch = _log(rng, 1, 16)
        hi = _log(rng, 33, 8192 // batch)
        case.update(batch=batch, new_lo=max(1, int(hi * rng.uniform(0.05, 1.0))), new_hi=hi, past_lo=0, past_hi=_log(rng, 1, 2048))
    if kind == "plan":
        return dict(case, batch=_log(rng, case["batch"], 300), forget=rng.choice((0.0, 0.3)))
    heads, kv = rng.choice(HEADS)
    dim = rng.choice((128, 64))
    return dict(case, dtype=rng.choice(("fp16", "bf16")), heads=heads, kv_heads=kv, dim=dim, rotary=rng.choice((dim, dim, dim // 2, dim // 4)),
                interleaved=rng.random() < 0.4)


# ---------------------------------------------------------------------------------------------- sizes
def _spaced(lo, hi, n):
    """n whole numbers from lo to hi, evenly spaced in the logarithm of their successors."""
    if n == 1:
        return [hi]
    return [round((lo + 1) * ((hi + 1) / (lo + 1)) ** (i / (n - 1))) - 1 for i in range(n)]


def _lengths(case):
    """New tokens and tokens in the cache before them, of every sequence: the longest prompts lie behind the shortest contexts."""
    return _spaced(case["new_lo"], case["new_hi"], case["batch"]), _spaced(case["past_lo"], case["past_hi"], case["batch"])[::-1]


def _counts(case):
    """Of a plan: new tokens of every sequence; every so many of them that have a context forget half of it instead."""
    new, past = _lengths(case)
    every = round(1 / case["forget"]) if case["forget"] else 0
    return [-(b // 2) if every and i % every == every - 1 and b > 1 else a for i, (a, b) in enumerate(zip(new, past))], past


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


def _needed(most):
    """The smallest power of two by which values up to `most` fit into e4m3, from 2^-24 to 2^7."""
    part, power = torch.frexp(most)                          # most / 448 = part 2^power / (0.875 * 2^9)
    return torch.ldexp(torch.ones_like(most), (power - 9 + (part > 0.875)).clamp(-24, 7)).where(most > 0, 2.0 ** -24)


def _codes(x, scale):
    return (x / scale).clamp(-MOST, MOST).to(E4M3)


def _pages(pool, case, g):
    """Pages in 8 bits of normal values, the blocks' sizes spread as those of different heads and places are, and their scales."""
    pages = torch.empty((pool, case["kv_heads"], case["page"] // BLOCK, BLOCK, case["dim"]), dtype=E4M3, device="cuda")
    scales = torch.empty(pages.shape[:3], dtype=torch.float16, device="cuda")
    for part in torch.arange(pool).split(max(1, (1 << 26) // pages[0].numel())):
        part = slice(int(part[0]), int(part[-1]) + 1)
        x = _randn(pages[part].shape, torch.float32, g)
        x *= torch.exp2(_randn(x.shape[:3], torch.float32, g) * 0.5)[..., None, None]
        scale = _needed(x.abs().amax(dim=(3, 4)))
        pages[part] = _codes(x, scale[..., None, None])
        scales[part] = scale
    return pages.view(pool, case["kv_heads"], case["page"], case["dim"]), scales


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
    state = dict(kind=case["kind"], table=table, lengths=length.int().cuda(), max_query=int(new.max()),
                 starts=None if case["new_hi"] == 1 else starts.cuda())
    for name in "kv":
        state[name], state[name + "_scales"] = _pages(pool, case, g)
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


def _prepare_plan(case, seed):
    g = _generator(seed, 1)
    order = torch.randperm(case["batch"], generator=torch.Generator().manual_seed(seed))
    counts, past = (torch.tensor(v, dtype=torch.int64)[order] for v in _counts(case))
    page = case["page"]
    have, want = (past + page - 1) // page, (past + counts + page - 1) // page
    width = int(torch.maximum(have, want).max()) + 1
    pool = int(torch.maximum(have, want).sum()) + 7
    pages = torch.randperm(pool, device="cuda", generator=g).int()
    used = int(have.sum())
    table = torch.full((case["batch"], width), -1, dtype=torch.int32, device="cuda")
    table[torch.arange(width, device="cuda")[None, :] < have.cuda()[:, None]] = pages[:used]
    free = torch.full((pool,), -1, dtype=torch.int32, device="cuda")
    free[:pool - used] = pages[used:]
    return dict(kind="plan", table=table, lengths=past.int().cuda(), counts=counts.int().cuda(), free=free, page=page,
                free_count=torch.tensor([pool - used], dtype=torch.int32, device="cuda"), rows=int(counts.clamp(min=0).sum()))


def _prepare_sample(case, seed):
    g = _generator(seed, 1)
    rows = case["rows"]
    state = dict(kind="sample", logits=(_randn((rows, case["vocab"]), torch.float32, g) * 2.5).to(DTYPES[case["dtype"]]),
                 uniform=torch.rand(rows, device="cuda", generator=g))
    settings = {n: case[n] for n in ("temperature", "top_k", "top_p", "min_p")}
    if case["mixed"]:                    # of every row its own, and each of them off in some rows
        pick = {"temperature": (0.0, 0.6, 0.8, 1.0, 1.3), "top_k": (0, 0, 1, 20, 50, 400), "top_p": (1.0, 1.0, 0.5, 0.9, 0.95),
                "min_p": (0.0, 0.0, 0.05, 0.1)}
        for n, values in pick.items():
            of = torch.randint(0, len(values), (rows,), device="cuda", generator=g)
            settings[n] = torch.tensor(values, dtype=torch.int32 if n == "top_k" else torch.float32, device="cuda")[of]
    return {**state, **settings}


def prepare(case, seed):
    return {"attention": _prepare_attention, "append": _prepare_append, "plan": _prepare_plan, "sample": _prepare_sample}[case["kind"]](case, seed)


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
    k, v = ((s[c].view(torch.uint8)[table].view(E4M3).float().unflatten(3, (-1, BLOCK)) * s[c + "_scales"][table].float()[..., None, None])
            .flatten(3, 4).transpose(1, 2).reshape(batch, kv, -1, dim) for c in "kv")
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


def _stored(pages, scales, rows, block, place, page, sub, first):
    """`rows` [tokens, kv, dim] into the blocks of 16 tokens that they belong to: row i at `place[i]` of block `block[i]`, which is block
    `sub` of page `page`; its first new token is at `first`, and the ones before it are scaled anew where the new ones need it."""
    blocks, kv, dim = page.shape[0], rows.shape[1], rows.shape[2]
    value = torch.zeros((blocks, BLOCK, kv, dim), dtype=torch.float32, device="cuda")
    value[block, place] = rows.float()
    fresh = torch.zeros((blocks, BLOCK), dtype=torch.bool, device="cuda")
    fresh[block, place] = True
    value = value.transpose(1, 2)                            # [blocks, kv, 16, dim]
    inside = pages.view(torch.uint8).view(pages.shape[0], kv, -1, BLOCK, dim)
    old, was = inside[page, :, sub], scales[page, :, sub].float()
    need = _needed(value.abs().amax(dim=(2, 3)))
    now = torch.where(first[:, None] > 0, torch.maximum(was, need), need)
    before = torch.arange(BLOCK, device="cuda") < first[:, None]
    again = _codes(old.view(E4M3).float() * was[..., None, None], now[..., None, None]).view(torch.uint8)
    code = torch.where(before[:, None, :, None], again, old)
    code = torch.where(fresh[:, None, :, None], _codes(value, now[..., None, None]).view(torch.uint8), code)
    inside[page, :, sub] = code
    scales[page, :, sub] = now.half()


def _plain_append(s):
    kv, page, dim = s["k"].shape[1:]
    qkv = s["qkv"].view(s["qkv"].shape[0], -1, dim)
    heads = qkv.shape[1] - 2 * kv
    seq, nth, position = _rows_of(s, qkv.shape[0])
    cos, sin = s["cos"][position], s["sin"][position]
    turned = _rotated(qkv[:, :heads + kv].float(), cos, sin, s["interleaved"]).to(qkv.dtype)
    begins = (nth == 0) | (position % BLOCK == 0)
    block = begins.cumsum(0) - 1
    at, of = position[begins], seq[begins]
    where = dict(block=block, place=position % BLOCK, page=s["table"][of, at // page].long(), sub=at % page // BLOCK, first=at % BLOCK)
    _stored(s["k"], s["k_scales"], turned[:, heads:], **where)
    _stored(s["v"], s["v_scales"], qkv[:, heads + kv:], **where)
    return {"q": turned[:, :heads].contiguous(), **{n: s[n] for n in ("k", "v", "k_scales", "v_scales")}}


def _plain_plan(s):
    page, table, lengths, counts, rows = s["page"], s["table"], s["lengths"].long(), s["counts"].long(), s["rows"]
    new = lengths + counts
    have, want = (lengths + page - 1) // page, (new + page - 1) // page
    column = torch.arange(table.shape[1], device="cuda")
    back = table[(column >= want[:, None]) & (column < have[:, None])]
    free, count = s["free"], s["free_count"].long()
    free[count + torch.arange(back.shape[0], device="cuda")] = back
    taken = (column >= have[:, None]) & (column < want[:, None])
    some = taken.sum()
    left = count + back.shape[0]
    table[taken] = free[left - 1 - torch.arange(some, device="cuda")]
    grown = counts.clamp(min=0)
    starts = torch.cat((torch.zeros(1, dtype=torch.int64, device="cuda"), grown.cumsum(0)))
    row = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(starts, row, right=True) - 1
    position = lengths[seq] + row - starts[seq]
    slots = table[seq, position // page].long() * page + position % page
    return {"table": table, "free": free, "lengths": new.int(), "starts": starts.int(), "positions": position.int(), "slots": slots,
            "free_count": (left - some).int(), "status": torch.zeros(1, dtype=torch.int32, device="cuda")}


def _plain_sample(s):
    x = s["logits"].double()
    rows, vocab = x.shape
    column = lambda n: s[n].double()[:, None] if torch.is_tensor(s[n]) else torch.full((rows, 1), float(s[n]), dtype=torch.float64, device="cuda")  # noqa: E731
    temperature, top_k, top_p, min_p = (column(n) for n in ("temperature", "top_k", "top_p", "min_p"))
    if not torch.is_tensor(s["top_p"]):                      # settings are fp32 numbers
        temperature, top_p, min_p = (t.float().double() for t in (temperature, top_p, min_p))
    ordered, index = torch.sort(s["logits"], dim=-1, descending=True, stable=True)
    top = ordered[:, :1].double()
    greedy = temperature <= 0
    weight = ((x - top) / torch.where(greedy, 1.0, temperature)).exp_()
    down = weight.gather(1, index)
    place = torch.arange(vocab, device="cuda")[None]
    inside = place < torch.where(top_k > 0, top_k, vocab)
    sums = torch.where(inside, down, 0.0).cumsum(dim=1)
    # an entry stays while those before it do not reach top_p of the whole
    inside &= (sums - down < top_p * sums[:, -1:]) | (top_p >= 1)
    inside &= down >= min_p
    inside[:, 0] = True
    inside &= (place == 0) | ~greedy
    kept = torch.zeros_like(inside).scatter_(1, index, inside)
    weight = weight.masked_fill_(~kept, 0.0)
    sums = weight.cumsum(dim=1)
    total = sums[:, -1:]
    token = (sums <= s["uniform"].double()[:, None] * total).sum(dim=1, keepdim=True).clamp(max=vocab - 1)
    return {"token": token[:, 0].int(), "logprob": (weight.gather(1, token) / total).log()[:, 0].float()}


def run(state):
    s = state
    if not own:
        return {"attention": _plain_attention, "append": _plain_append, "plan": _plain_plan, "sample": _plain_sample}[s["kind"]](s)
    from relax_b200 import ops

    if s["kind"] == "attention":
        return ops.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"], starts=s["starts"], max_query=s["max_query"],
                                   causal=s["causal"], window=s["window"], cap=s["cap"], slopes=s["slopes"], prefix=s["prefix"],
                                   k_scales=s["k_scales"], v_scales=s["v_scales"])
    if s["kind"] == "append":
        q = ops.paged_rope_append(s["qkv"], s["cos"], s["sin"], s["k"], s["v"], s["table"], s["lengths"], starts=s["starts"],
                                  interleaved=s["interleaved"], k_scales=s["k_scales"], v_scales=s["v_scales"])
        return {"q": q, **{n: s[n] for n in ("k", "v", "k_scales", "v_scales")}}
    if s["kind"] == "plan":
        r = ops.paged_plan(s["table"], s["lengths"], s["counts"], s["free"], s["free_count"], s["page"], s["rows"])
        return {"table": s["table"], "free": s["free"], "lengths": r.lengths, "starts": r.starts, "positions": r.positions, "slots": r.slots,
                "free_count": r.free_count, "status": r.status}
    r = ops.sample_tokens(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
    return {"token": r.token, "logprob": r.logprob}


# ---------------------------------------------------------------------------------------------- what a pass must do
def work(case):
    if case["kind"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (4 if case["dtype"] == "fp32" else 2) + case["rows"] * 28, "flops": 6 * n}
    page = case["page"]
    if case["kind"] == "plan":
        counts, past = _counts(case)
        moved = sum(abs(-(-(a + b) // page) + -b // page) for a, b in zip(counts, past))
        rows = sum(max(a, 0) for a in counts)
        return {"bytes": 16 * case["batch"] + 8 * moved + 12 * rows, "flops": 4 * rows + 8 * case["batch"]}
    new, past = _lengths(case)
    tokens = sum(new)
    pages = sum(-(-(a + b) // page) for a, b in zip(new, past))
    around = 4 * (pages + 2 * case["batch"])
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "append":
        blocks = sum((b + a - 1) // BLOCK - b // BLOCK + 1 for a, b in zip(new, past))
        turned = (heads + kv) * case["rotary"]
        return {"bytes": tokens * (2 * (heads + 2 * kv) * dim + 2 * heads * dim + 2 * kv * dim + 4 * case["rotary"]) + 8 * kv * blocks + around,
                "flops": tokens * (3 * turned + 4 * kv * dim)}
    counts = [_visible(case, a, b) for a, b in zip(new, past)]
    pairs, keys = sum(c[0] for c in counts), sum(c[1] for c in counts)
    return {"bytes": 4 * dim * tokens * heads + (2 * dim + 4 / BLOCK) * keys * kv + around, "flops": 4 * dim * heads * pairs}


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
            if h % group == 0:
                keys, values = (s[c].view(torch.uint8)[pages, h // group].view(E4M3).double().reshape(-1, case["dim"])
                                * s[c + "_scales"][pages, h // group].double().flatten().repeat_interleave(BLOCK)[:, None] for c in "kv")
                keys, values = keys[:length], values[:length]
            x = s["q"][rows, h].double() @ keys.T / math.sqrt(case["dim"])
            if case["cap"]:
                x = case["cap"] * torch.tanh(x / case["cap"])
            if case["slopes"]:
                x = x - 2.0 ** (-8.0 * (h + 1) / heads) * (i - j).abs()
            if case["causal"]:
                x = x.masked_fill(hidden, -math.inf)
            result[rows, h] = torch.softmax(x, dim=1) @ values
    return result


def _to_e4m3(x):
    """To the nearest of the format's numbers, in 64 bits: steps of 2^-3 of the leading bit's place, of 2^-9 below 2^-6."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-MOST, MOST)


def _exact_append(case, s):
    """Pair (a, b) at position t as the complex number a + ib times exp(i t w); then block by block of every sequence."""
    kv, page, dim, half = case["kv_heads"], case["page"], case["dim"], case["rotary"] // 2
    cos, sin = s["cos"].double(), s["sin"].double()
    codes = {c: s[c].double() for c in "kv"}
    scales = {c: s[c + "_scales"].double() for c in "kv"}
    qkv = s["qkv"].double().view(-1, case["heads"] + 2 * kv, dim)
    q = torch.empty((qkv.shape[0], case["heads"], dim), dtype=torch.float64, device="cuda")
    starts = s["starts"].tolist() if s["starts"] is not None else list(range(case["batch"] + 1))
    table = s["table"].tolist()
    for b, length in enumerate(s["lengths"].tolist()):
        new = starts[b + 1] - starts[b]
        first = length - new
        at = torch.arange(first, length, device="cuda")
        x = qkv[starts[b]:starts[b + 1]].clone()
        part = x[:, : case["heads"] + kv, : 2 * half]
        pairs = part.unflatten(-1, (half, 2)) if case["interleaved"] else part.unflatten(-1, (2, half)).transpose(-1, -2)
        turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * torch.complex(cos[at], sin[at])[:, None])
        part.copy_(turned.flatten(-2) if case["interleaved"] else turned.transpose(-1, -2).flatten(-2))
        q[starts[b]:starts[b + 1]] = x[:, : case["heads"]]
        for block in range(first // BLOCK, (length - 1) // BLOCK + 1):
            lo, hi = max(first, block * BLOCK), min(length, (block + 1) * BLOCK)
            where, offset = table[b][block * BLOCK // page], block * BLOCK % page
            for c, h0 in (("k", case["heads"]), ("v", case["heads"] + kv)):
                # (what a 16-bit cache would hold)
                y = x[lo - first:hi - first, h0:h0 + kv].to(DTYPES[case["dtype"]]).double().transpose(0, 1)
                scale = torch.exp2(torch.ceil(torch.log2(y.abs().amax(dim=(1, 2)) / MOST)).clamp(-24, 7))
                was = scales[c][where, :, offset // BLOCK].clone()
                if lo % BLOCK:
                    scale = torch.maximum(scale, was)
                    earlier = codes[c][where, :, offset:offset + lo % BLOCK]
                    codes[c][where, :, offset:offset + lo % BLOCK] = _to_e4m3(earlier * (was / scale)[:, None, None])
                codes[c][where, :, offset + lo % BLOCK:offset + lo % BLOCK + hi - lo] = _to_e4m3(y / scale[:, None, None])
                scales[c][where, :, offset // BLOCK] = scale
    return {"q": q, "k": codes["k"], "v": codes["v"], "k_scales": scales["k"], "v_scales": scales["v"]}


def _exact_sample(case, s):
    """Row by row: the kept entries as a set, in the order of their logits, then a walk along the indices."""
    tokens, logs = [], []
    of = lambda n, i: s[n][i].item() if torch.is_tensor(s[n]) else torch.tensor(s[n], dtype=torch.float32).item()  # noqa: E731
    for i in range(case["rows"]):
        x = s["logits"][i].double()
        temperature, top_k, top_p, min_p = (of(n, i) for n in ("temperature", "top_k", "top_p", "min_p"))
        order = torch.argsort(s["logits"][i].float(), descending=True, stable=True)
        if temperature <= 0:
            order = order[:1]
        elif top_k > 0:
            order = order[: int(top_k)]
        p = torch.softmax(x[order] / (temperature if temperature > 0 else 1.0), dim=0)
        if top_p < 1:
            n = int(torch.searchsorted(p.cumsum(0), torch.tensor([top_p], dtype=torch.float64, device="cuda"))) + 1
            order, p = order[:max(n, 1)], p[:max(n, 1)]
        n = max(1, int((p >= min_p * p[0]).sum()))
        by_index, back = torch.sort(order[:n])
        share = (p[:n] / p[:n].sum())[back]
        at = int(torch.searchsorted(share.cumsum(0), s["uniform"][i].double().view(1), right=True).clamp(max=n - 1))
        tokens.append(by_index[at])
        logs.append(share[at].log())
    return {"token": torch.stack(tokens).int(), "logprob": torch.stack(logs)}


def exact(case, seed):
    if case["kind"] == "plan":
        return None                      # whole numbers, all of them
    s = prepare(case, seed)
    return {"attention": _exact_attention, "append": _exact_append, "sample": _exact_sample}[case["kind"]](case, s)
