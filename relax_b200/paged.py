"""A q4f16 decoder over a paged key-value cache: prompts of any lengths in one call, then a token for every sequence at a time, with the
log probabilities of what was chosen.

What runs between the quantised matmuls is this library's: norm, SwiGLU and embedding as in :mod:`relax_b200.decoder`; rotary positions and
the append to the pages, attention over the pages, log probabilities (:mod:`relax_b200.ops`).  Key heads may be fewer than query heads,
sequences have lengths of their own, and a call takes any mixture of prompts, parts of prompts and single tokens.

    python -m relax_b200.paged --layers 4 --tokens 16        # random weights: two prompts, greedy tokens and their log probabilities
"""
from __future__ import annotations

import argparse
import dataclasses
import math
import operator

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
    scaling: dict | None = None        # see rope_tables

    def __post_init__(self):
        if self.heads % self.kv_heads or self.head_dim not in (64, 128):
            raise ValueError("heads is a multiple of kv_heads, head_dim is 64 or 128")


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


class PagedCache:
    """Pages of all layers and the tables of the sequences in them: ``batch`` places for sequences, each up to ``max_tokens`` long, over
    ``pages`` pages that they share."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, page_size: int, pages: int, batch: int, max_tokens: int,
                 dtype=torch.float16, device="cuda"):
        self.page_size, self.pages, self.device = page_size, pages, torch.device(device)
        shape = (pages, kv_heads, page_size, head_dim)
        self.k = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(layers)]
        self.v = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(layers)]
        self.max_tokens, self.width = max_tokens, -(-max_tokens // page_size)
        self.table_host = np.full((batch, self.width), -1, np.int32)
        self.lengths_host = np.zeros(batch, np.int32)
        self.free = list(range(pages - 1, -1, -1))

    def length(self, seq: int) -> int:
        """Tokens of a sequence.  (A negative number names no place: it would be another name for one of the last.)"""
        if not 0 <= seq < len(self.lengths_host):
            raise IndexError(f"place {seq} of the cache: there are {len(self.lengths_host)}")
        return int(self.lengths_host[seq])

    def extend(self, seq: int, tokens: int) -> None:
        """Room for `tokens` more of sequence `seq`; raises, and changes nothing, where the table or the pool has none."""
        length = self.length(seq)
        have, want = -(-length // self.page_size), -(-(length + tokens) // self.page_size)
        if tokens < 0 or length + tokens > self.max_tokens:
            raise ValueError(f"sequence {seq} of {length} tokens cannot grow by {tokens}: at most {self.max_tokens}")
        if want - have > len(self.free):
            raise MemoryError(f"{want - have} pages wanted, {len(self.free)} free")
        for i in range(have, want):
            self.table_host[seq, i] = self.free.pop()
        self.lengths_host[seq] += tokens

    def shrink(self, seq: int, tokens: int) -> None:
        """Forgets the last `tokens` of a sequence and gives back the pages that only they were in."""
        have = self.length(seq)
        keep = have - tokens
        if not 0 <= keep <= have:
            raise ValueError(f"sequence {seq} has {have} tokens: {tokens} of them cannot be forgotten")
        for i in range(-(-keep // self.page_size), -(-have // self.page_size)):
            self.free.append(int(self.table_host[seq, i]))
            self.table_host[seq, i] = -1
        self.lengths_host[seq] = keep

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
        self.cache = PagedCache(len(layers), cfg.kv_heads, cfg.head_dim, cfg.page_size, pages, batch, max_tokens, device=device)
        self.cos, self.sin = rope_tables(max_tokens, cfg.rotary, cfg.theta, cfg.scaling, device)

    def _stream(self):
        return torch.cuda.current_stream(self.device).cuda_stream

    def _norm(self, x, delta, weight, out):
        _lib.check(self.L.b200_rmsnorm(x.data_ptr(), None if delta is None else delta.data_ptr(), weight.data_ptr(), out.data_ptr(), x.shape[0],
                                       x.shape[1], self.cfg.eps, self._stream()))
        return out

    def forward(self, seqs, tokens, every: bool = False) -> torch.Tensor:
        """Takes `tokens[i]` (a list) as the next tokens of sequence `seqs[i]`: their keys and values go to the cache; the logits of the last
        of each, or with `every` of all of them, come back, fp16 [rows, vocab].  A call that raises leaves the sequences as they were."""
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
        cfg = self.cfg
        with torch.cuda.device(self.device):
            table, lengths = self.cache.tables(seqs)
            ids = torch.tensor(ids, dtype=torch.int32, device=self.device)
            T, H, f16 = ids.shape[0], cfg.hidden, dict(dtype=torch.float16, device=self.device)
            longest = max(counts)
            starts = None if longest == 1 else torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device=self.device)
            x, h, act = torch.empty((T, H), **f16), torch.empty((T, H), **f16), torch.empty((T, cfg.inter), **f16)
            _lib.check(self.L.b200_embed_rows(self.embed.data_ptr(), ids.data_ptr(), x.data_ptr(), T, H, self.embed.shape[0], self._stream()))
            delta = None
            for i, w in enumerate(self.layers):
                qkv = ops.q4f16_matmul(self._norm(x, delta, w["norm1"], h), *w["qkv"])
                q = ops.paged_rope_append(qkv, self.cos, self.sin, self.cache.k[i], self.cache.v[i], table, lengths, starts=starts,
                                          interleaved=cfg.interleaved)
                a = ops.paged_attention(q, self.cache.k[i], self.cache.v[i], table, lengths, starts=starts, max_query=longest, window=cfg.window,
                                        cap=cfg.cap)
                delta = ops.q4f16_matmul(a.view(T, -1), *w["o"])
                gu = ops.q4f16_matmul(self._norm(x, delta, w["norm2"], h), *w["gu"])
                _lib.check(self.L.b200_silu_mul(gu.data_ptr(), act.data_ptr(), T, cfg.inter, self._stream()))
                delta = ops.q4f16_matmul(act, *w["down"])
            self._norm(x, delta, self.final_norm, h)
            rows = h if every else h[torch.tensor(np.cumsum(counts) - 1, device=self.device)]
            return self._head(rows.contiguous())

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
    ap = argparse.ArgumentParser(description="Greedy tokens of a random q4f16 model over a paged cache")
    for name, value in (("layers", 4), ("hidden", 1024), ("heads", 8), ("kv-heads", 2), ("inter", 2816), ("vocab", 32000), ("tokens", 16), ("page-size", 16)):
        ap.add_argument(f"--{name}", type=int, default=value)
    a = ap.parse_args(argv)
    cfg = PagedConfig(hidden=a.hidden, heads=a.heads, kv_heads=a.kv_heads, inter=a.inter, layers=a.layers, vocab=a.vocab, page_size=a.page_size)
    g = torch.Generator(device="cuda").manual_seed(1)
    embed = torch.randn((cfg.vocab, cfg.hidden), dtype=torch.float16, device="cuda", generator=g) * 0.02
    model = PagedDecoder(cfg, [synth_layer(cfg, i) for i in range(cfg.layers)], embed, torch.ones(cfg.hidden, dtype=torch.float16, device="cuda"), embed,
                         batch=2, max_tokens=256)
    prompts = [list(range(5, 42)), [7, 9, 11]]
    for prompt, tokens, logprobs, entropies in zip(prompts, *model.generate(prompts, a.tokens)):
        print(f"prompt of {len(prompt)}:")
        for t, p, e in zip(tokens, logprobs, entropies):
            print(f"  {t:6d}  log p {p:8.4f}  entropy {e:7.4f}")
    print("score of the first prompt:", [round(v, 3) for v in model.score(0, prompts[0]).tolist()][:8], "...")


if __name__ == "__main__":
    main()
