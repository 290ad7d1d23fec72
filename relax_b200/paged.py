"""A q4f16 decoder over a paged key-value cache: prompts of any lengths in one call, then a token for every sequence at a time, with the
log probabilities of what was chosen.

What runs between the quantised matmuls is this library's: norm, SwiGLU and embedding as in :mod:`relax_b200.decoder`; rotary positions and
the append to the pages, attention over the pages, log probabilities (:mod:`relax_b200.ops`).  Key heads may be fewer than query heads,
sequences have lengths of their own, and a call takes any mixture of prompts, parts of prompts and single tokens.  Keys and values are held in 16
bits or in 8 (``cache_bits``).  :meth:`PagedDecoder.sample` draws tokens without the host between them: pages and rows planned, tokens drawn on the
device, a step one captured graph.

    python -m relax_b200.paged --layers 4 --tokens 16        # random weights: two prompts, greedy tokens and their log probabilities
    python -m relax_b200.paged --cache-bits 8 --temperature 0.8 --top-k 50 --top-p 0.9
"""
from __future__ import annotations

import argparse
import dataclasses
import math
import operator
import threading

import numpy as np
import torch

from . import _lib, ops, synth


@dataclasses.dataclass
class PagedConfig:
    hidden: int = 4096
    heads: int = 32
    kv_heads: int = 8
    inter: int = 11008
    layers: int = 32
    vocab: int = 32000
    eps: float = 1e-5
    theta: float = 10000.0
    head_dim: int = 128
    rotary: int = 128                  # values of a head that are turned
    interleaved: bool = False
    page_size: int = 16
    window: int = 0                    # tokens a row sees, itself among them (0: all before it)
    cap: float = 0.0                   # of the attention scores (0: none)
    cache_bits: int = 16               # of a key's or value's number in the pages; 8: e4m3 with a scale for 16 tokens of a head
    scaling: dict | None = None        # see rope_tables

    def __post_init__(self):
        if self.heads % self.kv_heads or self.head_dim not in (64, 128):
            raise ValueError("heads is a multiple of kv_heads, head_dim is 64 or 128")
        if self.cache_bits not in (8, 16):
            raise ValueError(f"cache_bits is 8 or 16, got {self.cache_bits}")


def rope_tables(positions: int, rotary: int, theta: float = 10000.0, scaling: dict | None = None, device="cuda"):
    """cos and sin, fp32 [positions, rotary / 2], formed in 64 bits.  ``scaling`` for contexts longer than a model was trained on:

    ``{"kind": "linear", "factor": f}``    positions divided by f
    ``{"kind": "base", "factor": f}``      theta times f^(rotary / (rotary - 2)): the slowest pair as if divided by f, the fastest as it was
    ``{"kind": "parts", "factor": f, "original": n, "low": a, "high": b}``  pairs that turn less than a times in n positions divided by f,
                                           those that turn more than b times kept, a straight line between
    and with any of them ``"magnitude": m``, a factor on both tables."""
    pair = np.arange(rotary // 2, dtype=np.float64)
    frequency = theta ** (-2.0 * pair / rotary)
    position = np.arange(positions, dtype=np.float64)
    scaling = dict(scaling or {})
    kind, magnitude = scaling.pop("kind", None), scaling.pop("magnitude", 1.0)
    if kind == "linear":
        position = position / scaling.pop("factor")
    elif kind == "base":
        if rotary <= 2:
            raise ValueError("a changed base needs more than one pair")
        frequency = (theta * scaling.pop("factor") ** (rotary / (rotary - 2))) ** (-2.0 * pair / rotary)
    elif kind == "parts":
        turns = scaling.pop("original") * frequency / (2 * math.pi)
        low, high = scaling.pop("low", 1.0), scaling.pop("high", 4.0)
        if not low < high:
            raise ValueError("low has to be less than high")
        kept = np.clip((turns - low) / (high - low), 0.0, 1.0)
        frequency = frequency * (kept + (1.0 - kept) / scaling.pop("factor"))
    elif kind is not None:
        raise ValueError(f"unknown scaling {kind!r}: linear, base or parts")
    if scaling:
        raise ValueError(f"unknown entries of scaling: {sorted(scaling)}")
    angle = position[:, None] * frequency[None, :]
    return tuple(torch.from_numpy((f(angle) * magnitude).astype(np.float32)).to(device).contiguous() for f in (np.cos, np.sin))


_pool = threading.RLock()              # one call at a time takes pages of a cache or gives them back (no cache's own: caches are copied and pickled)


class PagedCache:
    """Pages of all layers and the tables of the sequences in them: ``batch`` places for sequences, each up to ``max_tokens`` long, over
    ``pages`` pages that they share."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, page_size: int, pages: int, batch: int, max_tokens: int,
                 dtype=torch.float16, device="cuda"):
        self.page_size, self.pages, self.device = page_size, pages, torch.device(device)
        shape = (pages, kv_heads, page_size, head_dim)
        self.k = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(layers)]
        self.v = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(layers)]
        self.scales = [{}] * layers             # what the operators take beside the pages
        if dtype is torch.float8_e4m3fn:
            blocks = (pages, kv_heads, page_size // 16)
            self.scales = [{n: torch.ones(blocks, dtype=torch.float16, device=device) for n in ("k_scales", "v_scales")} for _ in range(layers)]
        self.max_tokens, self.width = max_tokens, -(-max_tokens // page_size)
        self.table_host = np.full((batch, self.width), -1, np.int32)
        self.lengths_host = np.zeros(batch, np.int32)
        self.free = list(range(pages - 1, -1, -1))
        self.held = set()                       # places of calls that keep their tables on the device

    def length(self, seq: int) -> int:
        """Tokens of a sequence.  (A negative number names no place: it would be another name for one of the last.)"""
        if not 0 <= seq < len(self.lengths_host):
            raise IndexError(f"place {seq} of the cache: there are {len(self.lengths_host)}")
        return int(self.lengths_host[seq])

    def _not_held(self, seq: int) -> int:
        length = self.length(seq)
        if seq in self.held:
            raise ValueError(f"place {seq} of the cache is in use by a call that has not returned")
        return length

    def extend(self, seq: int, tokens: int) -> None:
        """Room for `tokens` more of sequence `seq`; raises, and changes nothing, where the table or the pool has none."""
        with _pool:
            length = self._not_held(seq)
            have, want = -(-length // self.page_size), -(-(length + tokens) // self.page_size)
            if tokens < 0 or length + tokens > self.max_tokens:
                raise ValueError(f"sequence {seq} of {length} tokens cannot grow by {tokens}: at most {self.max_tokens}")
            if want - have > len(self.free):
                raise MemoryError(f"{want - have} pages wanted, {len(self.free)} free")
            for i in range(have, want):
                self.table_host[seq, i] = self.free.pop()
            self.lengths_host[seq] += tokens

    def shrink(self, seq: int, tokens: int) -> None:
        """Forgets the last `tokens` of a sequence and gives back the pages that only they were in.  In 8 bits a block of 16 of which some are left keeps
        the scale that the forgotten ones may have raised, and the rounding of its codes to it: 2^-10 of that scale at most."""
        with _pool:
            have = self._not_held(seq)
            keep = have - tokens
            if not 0 <= keep <= have:
                raise ValueError(f"sequence {seq} has {have} tokens: {tokens} of them cannot be forgotten")
            for i in range(-(-keep // self.page_size), -(-have // self.page_size)):
                self.free.append(int(self.table_host[seq, i]))
                self.table_host[seq, i] = -1
            self.lengths_host[seq] = keep

    def hold(self, tokens) -> list:
        """Takes the places 0 .. , which have to be empty, for sequences of up to ``tokens[i]`` each, and pages for all of them, which it returns: for a
        call whose tables are its own.  Nobody else gets the places or the pages before :meth:`give_back`.  Raises, and changes nothing, where
        there is no room."""
        with _pool:
            if any([self.length(s) for s in range(len(tokens))]) or not self.held.isdisjoint(range(len(tokens))):
                raise ValueError("the first places of the cache are in use")
            if max(tokens, default=0) > self.max_tokens:
                raise ValueError(f"a sequence of {max(tokens)} tokens: at most {self.max_tokens}")
            pages = sum(-(-n // self.page_size) for n in tokens)
            if pages > len(self.free):
                raise MemoryError(f"{pages} pages wanted, {len(self.free)} free")
            taken = self.free[len(self.free) - pages:]
            del self.free[len(self.free) - pages:]
            self.held.update(range(len(tokens)))
            self.lengths_host[:len(tokens)] = tokens
            return taken

    def give_back(self, places: int, pages) -> None:
        """The places 0 .. places - 1 are empty again, and the pages free."""
        with _pool:
            self.free.extend(pages)
            self.held.difference_update(range(places))
            self.lengths_host[:places] = 0

    def release(self, seq: int) -> None:
        """Gives the pages of a sequence back."""
        self.shrink(seq, self.length(seq))

    def tables(self, seqs):
        """Page table and lengths of these sequences on the device, as the operators take them; the table as wide as the longest needs."""
        lengths = self.lengths_host[seqs]
        width = max(1, -(-int(lengths.max()) // self.page_size))
        return (torch.from_numpy(np.ascontiguousarray(self.table_host[seqs, :width])).to(self.device),
                torch.from_numpy(np.ascontiguousarray(lengths)).to(self.device))


def synth_layer(cfg: PagedConfig, seed: int, device="cuda") -> dict:
    """Random weights of one layer, as small as a trained model's."""
    H, D = cfg.hidden, cfg.head_dim
    shapes = {"qkv": ((cfg.heads + 2 * cfg.kv_heads) * D, H), "o": (H, cfg.heads * D), "gu": (2 * cfg.inter, H), "down": (H, cfg.inter)}
    layer = {}
    for j, (name, (n, k)) in enumerate(shapes.items()):
        wq, scales = synth.make_weights_torch(n, k, seed * 16 + j, device)
        layer[name] = (wq, scales * 0.1)
    for name in ("norm1", "norm2"):
        layer[name] = torch.ones(H, dtype=torch.float16, device=device)
    return layer


class PagedDecoder:
    """Weights, cache and the kernel sequence of a call.  ``layers``: a list of dicts as :func:`synth_layer` makes them; ``embed`` fp16
    [vocab, hidden]; ``lm_head`` fp16 [vocab, hidden]."""

    def __init__(self, cfg: PagedConfig, layers, embed, final_norm, lm_head, batch: int, max_tokens: int, pages: int | None = None, device="cuda"):
        self.cfg, self.layers, self.embed, self.final_norm, self.lm_head = cfg, layers, embed, final_norm, lm_head
        self.device = torch.device(device)
        self.L = _lib.lib()
        pages = batch * -(-max_tokens // cfg.page_size) if pages is None else pages
        self.cache = PagedCache(len(layers), cfg.kv_heads, cfg.head_dim, cfg.page_size, pages, batch, max_tokens,
                                dtype=torch.float16 if cfg.cache_bits == 16 else torch.float8_e4m3fn, device=device)
        self.cos, self.sin = rope_tables(max_tokens, cfg.rotary, cfg.theta, cfg.scaling, device)

    def _stream(self):
        return torch.cuda.current_stream(self.device).cuda_stream

    def _norm(self, x, delta, weight, out):
        _lib.check(self.L.b200_rmsnorm(x.data_ptr(), None if delta is None else delta.data_ptr(), weight.data_ptr(), out.data_ptr(), x.shape[0],
                                       x.shape[1], self.cfg.eps, self._stream()))
        return out

    def forward(self, seqs, tokens, every: bool = False) -> torch.Tensor:
        """Takes `tokens[i]` (a list) as the next tokens of sequence `seqs[i]`: their keys and values go to the cache; the logits of the last
        of each, or with `every` of all of them, come back, fp16 [rows, vocab].  A call that raises leaves the sequences as they were: their lengths and
        pages, and in 16 bits their keys and values.  In 8 bits it is as if the new tokens had come and been forgotten (:meth:`PagedCache.shrink`)."""
        counts = [len(t) for t in tokens]
        if len(seqs) != len(tokens) or len(set(seqs)) != len(seqs) or min(counts, default=0) < 1:
            raise ValueError("every sequence once, with one token at least")
        ids = [operator.index(t) for ts in tokens for t in ts]
        if not 0 <= min(ids) <= max(ids) < self.embed.shape[0]:
            raise ValueError(f"tokens are 0 to {self.embed.shape[0] - 1}, got {min(ids)} to {max(ids)}")
        done = []
        try:
            for s, n in zip(seqs, counts):
                self.cache.extend(s, n)
                done.append((s, n))
            return self._forward(list(seqs), ids, counts, every)
        except BaseException:                       # (nothing may count that has no keys in every layer)
            for s, n in done:
                self.cache.shrink(s, n)
            raise

    def _forward(self, seqs, ids, counts, every: bool) -> torch.Tensor:
        with torch.cuda.device(self.device):
            table, lengths = self.cache.tables(seqs)
            ids = torch.tensor(ids, dtype=torch.int32, device=self.device)
            longest = max(counts)
            starts = None if longest == 1 else torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device=self.device)
            h = self._rows(ids, table, lengths, starts, longest)
            rows = h if every else h[torch.tensor(np.cumsum(counts) - 1, device=self.device)]
            return self._head(rows.contiguous())

    def _rows(self, ids, table, lengths, starts, longest: int, scratch=None) -> torch.Tensor:
        """The tokens `ids` (on the device) through all layers, the last norm included."""
        cfg = self.cfg
        T, H, f16 = ids.shape[0], cfg.hidden, dict(dtype=torch.float16, device=self.device)
        x, h, act = torch.empty((T, H), **f16), torch.empty((T, H), **f16), torch.empty((T, cfg.inter), **f16)
        _lib.check(self.L.b200_embed_rows(self.embed.data_ptr(), ids.data_ptr(), x.data_ptr(), T, H, self.embed.shape[0], self._stream()))
        delta = None
        for i, w in enumerate(self.layers):
            pages = (self.cache.k[i], self.cache.v[i], table, lengths)
            qkv = ops.q4f16_matmul(self._norm(x, delta, w["norm1"], h), *w["qkv"])
            q = ops.paged_rope_append(qkv, self.cos, self.sin, *pages, starts=starts, interleaved=cfg.interleaved, **self.cache.scales[i])
            a = ops.paged_attention(q, *pages, starts=starts, max_query=longest, window=cfg.window, cap=cfg.cap, scratch=scratch, **self.cache.scales[i])
            delta = ops.q4f16_matmul(a.view(T, -1), *w["o"])
            gu = ops.q4f16_matmul(self._norm(x, delta, w["norm2"], h), *w["gu"])
            _lib.check(self.L.b200_silu_mul(gu.data_ptr(), act.data_ptr(), T, cfg.inter, self._stream()))
            delta = ops.q4f16_matmul(act, *w["down"])
        self._norm(x, delta, self.final_norm, h)
        return h

    def _head(self, h):
        rows, vocab = h.shape[0], self.lm_head.shape[0]
        logits = torch.empty((rows, vocab), dtype=torch.float16, device=self.device)
        if rows > 16:                               # (the library's output projection takes up to 16 rows)
            return torch.matmul(h, self.lm_head.t(), out=logits)
        _lib.check(self.L.b200_lm_head(h.data_ptr(), self.lm_head.data_ptr(), logits.data_ptr(), None, None, rows, vocab, h.shape[1], 0,
                                       self._stream()))
        return logits

    def generate(self, prompts, new_tokens: int, top: int = 1):
        """Greedy tokens behind the prompts: (tokens, their log probabilities, entropies), each [sequences][new_tokens].  Uses places 0 .. of the
        cache, which have to be empty, and gives their pages back.  `top` changes nothing (a greedy step takes the likeliest) and is there for
        callers that give it; alternatives come from :func:`relax_b200.ops.token_logprobs`."""
        seqs = list(range(len(prompts)))
        if any(self.cache.length(s) for s in seqs):
            raise ValueError("the first places of the cache are in use")
        chosen, logprobs, entropies = [], [], []
        try:
            for step in range(new_tokens):
                logits = self.forward(seqs, prompts if step == 0 else [[t] for t in chosen[-1]])
                none = torch.zeros(len(seqs), dtype=torch.int32, device=self.device)
                said = ops.token_logprobs(logits, none, top=1)
                chosen.append(said.top_token[:, 0].tolist())
                logprobs.append(said.top_logprob[:, 0].tolist())
                entropies.append(said.entropy.tolist())
        finally:
            for s in seqs:
                self.cache.release(s)
        return tuple([[step[s] for step in v] for s in seqs] for v in (chosen, logprobs, entropies))

    def sample(self, prompts, new_tokens: int, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, seed: int = 0, uniform: torch.Tensor | None = None):
        """Drawn tokens behind the prompts: (tokens, logarithms of their shares among what could have come), each [sequences][new_tokens].  The
        settings are those of :func:`relax_b200.ops.sample_tokens`, numbers or tensors of one for each sequence; ``uniform`` (fp32 [new_tokens,
        sequences]) gives the random numbers, else they come from `seed`.

        Uses places 0 .. of the cache, which have to be empty, and leaves them so: the tables of the call are its own, on the device, over pages that
        nobody else gets while it runs.  A call that finds no room for all of it raises before it begins; one in which a row of logits holds a NaN or
        an infinity, so that nothing can be drawn, raises at its end."""
        n, cache = len(prompts), self.cache
        counts = [len(t) for t in prompts]
        ids = [operator.index(t) for ts in prompts for t in ts]
        if n == 0 or min(counts) < 1 or new_tokens < 0:
            raise ValueError("every prompt has one token at least")
        if not 0 <= min(ids) <= max(ids) < self.embed.shape[0]:
            raise ValueError(f"tokens are 0 to {self.embed.shape[0] - 1}, got {min(ids)} to {max(ids)}")
        most = [c + new_tokens - 1 if new_tokens else 0 for c in counts]     # (the last token drawn has no keys)
        pages = cache.hold(most)
        try:
            if new_tokens == 0:
                return [[] for _ in prompts], [[] for _ in prompts]
            with torch.cuda.device(self.device):
                if uniform is None:
                    uniform = torch.rand((new_tokens, n), device=self.device, generator=torch.Generator(device=self.device).manual_seed(seed))
                elif uniform.shape != (new_tokens, n) or uniform.dtype is not torch.float32 or uniform.device != self.embed.device or not uniform.is_contiguous():
                    raise ValueError(f"uniform is a contiguous fp32 tensor {(new_tokens, n)} on {self.embed.device}")
                return self._sample(counts, ids, max(most), pages, uniform, dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p))
        finally:
            cache.give_back(n, pages)

    def _sample(self, counts, ids, longest: int, pages, uniform, how):
        cache = self.cache
        new_tokens, n = uniform.shape
        i32 = dict(dtype=torch.int32, device=self.device)
        table = torch.full((n, -(-longest // cache.page_size)), -1, **i32)
        free, free_count = torch.tensor(pages, **i32), torch.tensor([len(pages)], **i32)
        lengths, ones = torch.zeros(n, **i32), torch.ones(n, **i32)
        tokens, logprobs = torch.empty((new_tokens, n), **i32), torch.empty((new_tokens, n), dtype=torch.float32, device=self.device)

        def plan(counts, rows):
            out = ops.paged_plan_buffers(n, rows, self.device)._replace(lengths=lengths, free_count=free_count)
            return ops.paged_plan(table, lengths, counts, free, free_count, cache.page_size, rows, cache.max_tokens, out=out)

        # the prompts
        p = plan(torch.tensor(counts, **i32), sum(counts))
        h = self._rows(torch.tensor(ids, **i32), table, lengths, p.starts if max(counts) > 1 else None, max(counts))
        drawn = ops.sample_tokens(self._head(h[p.starts[1:].long() - 1]), uniform[0], **how)
        tokens[0], logprobs[0] = drawn.token, drawn.logprob
        # the tokens behind them: what a step reads and writes lies where the graph expects it
        token, u, scratch = drawn.token, torch.empty(n, dtype=torch.float32, device=self.device), ops.paged_attention_scratch(self.device)

        def step():
            plan(ones, n)
            drawn = ops.sample_tokens(self._head(self._rows(token, table, lengths, None, 1, scratch)), u, **how)
            token.copy_(drawn.token)
            return drawn.logprob

        graph = None
        for i in range(1, new_tokens):
            u.copy_(uniform[i])
            if graph is None and 2 <= i < new_tokens - 1:            # (the first step prepares what a capture may not)
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, capture_error_mode="thread_local"):     # (other threads may go on with their calls)
                    held = step()
            if graph is None:
                logprobs[i] = step()
            else:
                graph.replay()
                logprobs[i] = held
            tokens[i] = token
        tokens = tokens.t().tolist()
        for s, of in enumerate(tokens):              # (the steps behind it went on from a token that nobody drew)
            if -1 in of:
                raise ValueError(f"nothing to draw for sequence {s} at its token {of.index(-1)}: its logits hold a NaN or an infinity, or exclude everything")
        return tokens, logprobs.t().tolist()

    def score(self, seq: int, tokens):
        """Log probability of every token of a text but its first, given those before it (sequence place `seq`, which has to be empty)."""
        if self.cache.length(seq):
            raise ValueError(f"place {seq} of the cache is in use")
        try:
            logits = self.forward([seq], [list(tokens)], every=True)
            want = torch.tensor(list(tokens[1:]) + [-1], dtype=torch.int32, device=self.device)
            return ops.token_logprobs(logits, want).logprob[:-1]
        finally:
            self.cache.release(seq)


def main(argv=None):
    ap = argparse.ArgumentParser(description="Tokens of a random q4f16 model over a paged cache")
    for name, value in (("layers", 4), ("hidden", 1024), ("heads", 8), ("kv-heads", 2), ("inter", 2816), ("vocab", 32000), ("tokens", 16), ("page-size", 16),
                        ("cache-bits", 16), ("top-k", 0), ("seed", 0)):
        ap.add_argument(f"--{name}", type=int, default=value)
    for name, value in (("temperature", 0.0), ("top-p", 1.0), ("min-p", 0.0)):
        ap.add_argument(f"--{name}", type=float, default=value, help="drawn tokens, with a temperature above 0" if name == "temperature" else None)
    a = ap.parse_args(argv)
    cfg = PagedConfig(hidden=a.hidden, heads=a.heads, kv_heads=a.kv_heads, inter=a.inter, layers=a.layers, vocab=a.vocab, page_size=a.page_size,
                      cache_bits=a.cache_bits)
    g = torch.Generator(device="cuda").manual_seed(1)
    embed = torch.randn((cfg.vocab, cfg.hidden), dtype=torch.float16, device="cuda", generator=g) * 0.02
    model = PagedDecoder(cfg, [synth_layer(cfg, i) for i in range(cfg.layers)], embed, torch.ones(cfg.hidden, dtype=torch.float16, device="cuda"), embed,
                         batch=2, max_tokens=256)
    prompts = [list(range(5, 42)), [7, 9, 11]]
    if a.temperature > 0:
        drawn = model.sample(prompts, a.tokens, a.temperature, a.top_k, a.top_p, a.min_p, a.seed)
        for prompt, tokens, logprobs in zip(prompts, *drawn):
            print(f"prompt of {len(prompt)}:")
            for t, p in zip(tokens, logprobs):
                print(f"  {t:6d}  log p {p:8.4f}")
        return
    for prompt, tokens, logprobs, entropies in zip(prompts, *model.generate(prompts, a.tokens)):
        print(f"prompt of {len(prompt)}:")
        for t, p, e in zip(tokens, logprobs, entropies):
            print(f"  {t:6d}  log p {p:8.4f}  entropy {e:7.4f}")
    print("score of the first prompt:", [round(v, 3) for v in model.score(0, prompts[0]).tolist()][:8], "...")


if __name__ == "__main__":
    main()
