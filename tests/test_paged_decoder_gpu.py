"""The decoder over the paged cache against the same model in 64 bits, and against itself: a prompt at once, in parts, token by token."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import oracle
from relax_b200 import ops, paged

pytestmark = pytest.mark.gpu


def model(**kw):
    cfg = paged.PagedConfig(**{**dict(hidden=512, heads=4, kv_heads=2, inter=768, layers=2, vocab=1000, page_size=16), **kw})
    g = torch.Generator(device="cuda").manual_seed(3)
    embed = torch.randn((cfg.vocab, cfg.hidden), dtype=torch.float16, device="cuda", generator=g) * 0.05
    layers = [paged.synth_layer(cfg, 10 + i) for i in range(cfg.layers)]
    for w in layers:                                            # (attention far from uniform)
        w["qkv"] = (w["qkv"][0], w["qkv"][1] * 6)
        w["norm1"] = (1 + 0.1 * torch.randn(cfg.hidden, device="cuda", generator=g)).half()
    return paged.PagedDecoder(cfg, layers, embed, torch.ones(cfg.hidden, dtype=torch.float16, device="cuda"), embed, batch=4, max_tokens=300)


def reference(m, tokens):
    """Logits of every token, in 64 bits over the dequantised weights."""
    cfg, D = m.cfg, m.cfg.head_dim
    group = cfg.heads // cfg.kv_heads
    x = m.embed.double().cpu().numpy()[tokens]
    norm = lambda v, w: v / np.sqrt((v * v).mean(axis=1, keepdims=True) + cfg.eps) * w.double().cpu().numpy()
    w64 = lambda w: oracle.c_dequantize(w[0].cpu().numpy(), w[1].cpu().numpy()).astype(np.float64)
    n, half = len(tokens), cfg.rotary // 2
    cos, sin = m.cos.double().cpu().numpy()[:n, None], m.sin.double().cpu().numpy()[:n, None]

    def turn(v):
        a, b = (v[..., 0:2 * half:2], v[..., 1:2 * half:2]) if cfg.interleaved else (v[..., :half], v[..., half:2 * half])
        p, q = a * cos - b * sin, b * cos + a * sin
        t = np.stack([p, q], axis=-1).reshape(*p.shape[:-1], 2 * half) if cfg.interleaved else np.concatenate([p, q], axis=-1)
        return np.concatenate([t, v[..., 2 * half:]], axis=-1)

    i, j = np.arange(n)[:, None], np.arange(n)[None]
    hidden = (j > i) | ((i - j >= cfg.window) if cfg.window else False)
    for w in m.layers:
        qkv = (norm(x, w["norm1"]) @ w64(w["qkv"]).T).reshape(n, -1, D)
        q, k, v = turn(qkv[:, :cfg.heads]), turn(qkv[:, cfg.heads:cfg.heads + cfg.kv_heads]), qkv[:, cfg.heads + cfg.kv_heads:]
        out = np.empty((n, cfg.heads, D))
        for h in range(cfg.heads):
            s = q[:, h] @ k[:, h // group].T / math.sqrt(D)
            if cfg.cap:
                s = cfg.cap * np.tanh(s / cfg.cap)
            s[hidden] = -np.inf
            p = np.exp(s - s.max(axis=1, keepdims=True))
            out[:, h] = p @ v[:, h // group] / p.sum(axis=1, keepdims=True)
        x = x + out.reshape(n, -1) @ w64(w["o"]).T
        gu = norm(x, w["norm2"]) @ w64(w["gu"]).T
        gate, up = gu[:, :cfg.inter], gu[:, cfg.inter:]
        x = x + gate / (1 + np.exp(-gate)) * up @ w64(w["down"]).T
    return norm(x, m.final_norm) @ m.lm_head.double().cpu().numpy().T


# fp16 between the kernels: the bound of the other decoder tests, 1e-2 of the tensor's scale
def near(got, want):
    got = got.double().cpu().numpy()
    assert np.isfinite(got).all() and np.abs(got - want).max() <= 1e-2 * np.abs(want).max(), np.abs(got - want).max() / np.abs(want).max()


@pytest.mark.parametrize("kw", [dict(), dict(kv_heads=4, page_size=32), dict(kv_heads=1, cap=20.0, interleaved=True, rotary=64), dict(window=9),
                                dict(heads=8, kv_heads=2, head_dim=64, rotary=32)])
def test_against_64_bits(cuda_lib, kw):
    m = model(**kw)
    rng = np.random.default_rng(1)
    texts = [rng.integers(0, m.cfg.vocab, n).tolist() for n in (1, 40, 17, 130)]
    want = [reference(m, t) for t in texts]
    # all prompts at once
    logits = m.forward([0, 1, 2, 3], texts, every=True)
    for got, w in zip(logits.split([len(t) for t in texts]), want):
        near(got, w)
    for s in range(4):
        m.cache.release(s)
    assert len(m.cache.free) == m.cache.pages
    # in parts that mix prompts, rests of prompts and single tokens; other places of the cache
    near(m.forward([2, 0], [texts[1][:20], texts[3][:100]]), np.stack([want[1][19], want[3][99]]))
    near(m.forward([1, 2, 0], [texts[2][:5], texts[1][20:39], texts[3][100:101]]), np.stack([want[2][4], want[1][38], want[3][100]]))
    near(m.forward([0, 2, 1], [[texts[3][101]], [texts[1][39]], [texts[2][5]]]), np.stack([want[3][101], want[1][39], want[2][5]]))


def test_generation_and_scores(cuda_lib):
    m = model()
    prompts = [[5, 6, 7, 8, 9, 10, 11], [3]]
    tokens, logprobs, entropies = m.generate(prompts, 6)
    for prompt, ts, ps, es in zip(prompts, tokens, logprobs, entropies):
        text = list(prompt)
        for t, p, e in zip(ts, ps, es):
            row = torch.from_numpy(reference(m, text)[-1])
            log = torch.log_softmax(row, dim=0)
            assert abs(float(log[t]) - p) < 0.05 and float(log.max()) - float(log[t]) < 0.05        # (greedy but for fp16's rounding)
            assert abs(float(-(log.exp() * log).sum()) - e) < 0.05
            text.append(t)
        scores = m.score(1, text)
        want = torch.log_softmax(torch.from_numpy(reference(m, text)), dim=1)[torch.arange(len(text) - 1), torch.tensor(text[1:])]
        assert scores.shape == (len(text) - 1,) and (scores.double().cpu() - want).abs().max() < 0.05
    assert len(m.cache.free) == m.cache.pages


def test_refusals_leave_the_cache_alone(cuda_lib):
    m = model()
    m.forward([0], [[1, 2, 3]])
    for seqs, tokens in (([0, 0], [[1], [2]]), ([0], [[]]), ([0, 1], [[1]]), ([1, 0], [[4], [5] * 400])):
        with pytest.raises(ValueError):
            m.forward(seqs, tokens)
    assert m.cache.lengths_host.tolist() == [3, 0, 0, 0] and len(m.cache.free) == m.cache.pages - 1
    with pytest.raises(ValueError):
        m.generate([[1]], 2)
    with pytest.raises(ValueError):
        m.score(0, [1, 2])
    near(m.forward([0], [[4]]), reference(m, [1, 2, 3, 4])[-1:])


def test_the_command(cuda_lib, capsys):
    paged.main(["--layers", "1", "--hidden", "256", "--heads", "2", "--kv-heads", "1", "--inter", "512", "--vocab", "500", "--tokens", "3"])
    out = capsys.readouterr().out
    assert out.count("log p") == 6 and "score" in out
