"""The decoder with keys and values in 8 bits, and tokens drawn without the host: against the same steps taken one by one."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from relax_b200 import ops, paged
from test_paged_decoder_gpu import model

pytestmark = pytest.mark.gpu


def by_hand(m, prompts, n, uniform, **how):
    """Drawn tokens by forward() and sample_tokens, tables on the host."""
    seqs = list(range(len(prompts)))
    tokens, logprobs, feed = [], [], prompts
    for i in range(n):
        drawn = ops.sample_tokens(m.forward(seqs, feed), uniform[i], **how)
        tokens.append(drawn.token.tolist())
        logprobs.append(drawn.logprob.tolist())
        feed = [[t] for t in tokens[-1]]
    for s in seqs:
        m.cache.release(s)
    return [list(t) for t in zip(*tokens)], [list(t) for t in zip(*logprobs)]


@pytest.mark.parametrize("kw", [dict(), dict(kv_heads=4, page_size=32), dict(kv_heads=1, cap=20.0, interleaved=True, rotary=64), dict(window=9),
                                dict(heads=8, kv_heads=2, head_dim=64, rotary=32)])
def test_eight_bits_stay_near_sixteen(cuda_lib, kw):
    """The same weights with both caches.  A number in 8 bits is off by 2^-4 of itself at most and by 0.026 on average, so attention's results are
    off by a few hundredths of the values' size; the logits of two layers stay within a tenth of theirs."""
    texts = [np.random.default_rng(1).integers(0, 1000, n).tolist() for n in (1, 40, 17, 130)]
    sixteen = model(**kw).forward([0, 1, 2, 3], texts, every=True).float()
    m = model(cache_bits=8, **kw)
    eight = m.forward([0, 1, 2, 3], texts, every=True).float()
    assert torch.isfinite(eight).all() and (eight - sixteen).abs().max() <= 0.1 * sixteen.abs().max()
    assert (eight - sixteen).norm() <= 0.05 * sixteen.norm()
    # the first token of a text sees itself alone, and its value's codes say so
    assert m.cache.k[0].dtype is torch.float8_e4m3fn and m.cache.scales[0]["k_scales"].shape == (m.cache.pages, m.cfg.kv_heads, m.cfg.page_size // 16)


@pytest.mark.parametrize("bits", (8, 16))
def test_a_text_in_parts_says_the_same(cuda_lib, bits):
    """Prompts at once and token by token.  In 8 bits a block's scale may grow under its first tokens, whose codes are then rounded again only where
    they fall below the format's smallest step: the caches are the same but for that and for the rounding of the matmuls."""
    m = model(cache_bits=bits)
    text = np.random.default_rng(2).integers(0, 1000, 50).tolist()
    whole = m.forward([0], [text], every=True).float()
    parts = torch.cat([m.forward([1], [text[a:b]], every=True).float() for a, b in ((0, 1), (1, 7), (7, 8), (8, 40), (40, 50))])
    assert (whole - parts).abs().max() <= 0.1 * whole.abs().max()


@pytest.mark.parametrize("bits", (8, 16))
@pytest.mark.parametrize("how", (dict(temperature=0.0), dict(temperature=0.9, top_k=20, top_p=0.9), dict(temperature=1.2, min_p=0.02)))
@pytest.mark.parametrize("lengths", ((5,), (1, 37, 16, 2)))
def test_drawn_tokens_are_those_of_the_single_steps(cuda_lib, bits, how, lengths):
    """The graph's steps and the host's run the same kernels on the same numbers: same tokens, same log probabilities."""
    m = model(cache_bits=bits)
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, 1000, n).tolist() for n in lengths]
    uniform = torch.rand((12, len(prompts)), device="cuda", generator=torch.Generator(device="cuda").manual_seed(4))
    want = by_hand(m, prompts, 12, uniform, **how)
    free = list(m.cache.free)
    got = m.sample(prompts, 12, uniform=uniform, **how)
    assert got[0] == want[0] and np.allclose(got[1], want[1], rtol=0, atol=1e-5)
    assert m.cache.free == free and not m.cache.lengths_host.any()
    assert m.sample(prompts, 12, uniform=uniform, **how) == got
    assert m.sample(prompts, 2, uniform=uniform[:2].contiguous(), **how)[0] == [t[:2] for t in got[0]]


def test_settings_of_their_own_and_seeds(cuda_lib):
    m = model(cache_bits=8)
    prompts = [[1, 2, 3], [4], [5, 6]]
    t = torch.tensor([0.0, 1.0, 2.0], device="cuda")
    k = torch.tensor([0, 1, 50], dtype=torch.int32, device="cuda")
    first = m.sample(prompts, 6, temperature=t, top_k=k, seed=1)
    greedy = m.sample(prompts, 6, temperature=0.0)
    assert first[0][:2] == greedy[0][:2] and first[1][0] == [0.0] * 6
    assert m.sample(prompts, 6, temperature=t, top_k=k, seed=1) == first and m.sample(prompts, 6, temperature=2.0, seed=2) != m.sample(prompts, 6, temperature=2.0, seed=3)
    assert m.sample(prompts, 0) == ([[], [], []], [[], [], []])


def test_refusals_leave_everything_as_it_was(cuda_lib):
    m = model(cache_bits=8)
    free = list(m.cache.free)
    for prompts, n, error in (([[]], 3, ValueError), ([], 3, ValueError), ([[1]], -1, ValueError), ([[1000]], 2, ValueError), ([[1] * 200], 102, ValueError)):
        with pytest.raises(error):
            m.sample(prompts, n)
    with pytest.raises(ValueError):
        m.sample([[1]], 3, uniform=torch.zeros(3, device="cuda"))
    m.forward([0], [[1, 2]])
    with pytest.raises(ValueError):
        m.sample([[1]], 3)
    m.cache.release(0)
    m.cache.free = m.cache.free[:2]
    with pytest.raises(MemoryError):
        m.sample([[1] * 20, [2]], 20)
    m.cache.free = free
    with pytest.raises(ValueError):
        paged.PagedConfig(cache_bits=4)


def test_the_command(cuda_lib, capsys):
    paged.main(["--layers", "1", "--hidden", "512", "--heads", "4", "--inter", "768", "--vocab", "500", "--tokens", "4", "--cache-bits", "8", "--temperature", "0.8",
                "--top-k", "20"])
    assert capsys.readouterr().out.count("log p") == 8
