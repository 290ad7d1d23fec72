"""PagedDecoder.sample beside other calls on the same cache."""
import threading

import pytest

torch = pytest.importorskip("torch")

from relax_b200 import ops
from test_paged_decoder_gpu import model

pytestmark = pytest.mark.gpu
PROMPTS = [[5, 6, 7, 8], list(range(40, 77))]


@pytest.mark.parametrize("bits", (8, 16))
def test_calls_in_the_middle_of_a_sample(cuda_lib, monkeypatch, bits):
    """forward() on another place between two steps gets other pages, and sample() none of the places in use: both say what they say alone."""
    m = model(cache_bits=bits)
    text = list(range(300, 390))
    alone = m.forward([3], [text])
    m.cache.release(3)
    want = m.sample(PROMPTS, 3, seed=1)
    free, drawn, between = list(m.cache.free), ops.sample_tokens, []

    def draw(*args, **how):
        out = drawn(*args, **how)
        if not between:
            between.append(None)
            between[0] = m.forward([3], [text])
            for call in (lambda: m.sample([[1]], 2), lambda: m.generate([[1]], 2), lambda: m.score(0, [1, 2]), lambda: m.forward([0], [[1]])):
                with pytest.raises(ValueError, match="in use"):
                    call()
            m.cache.release(3)
        return out

    monkeypatch.setattr(ops, "sample_tokens", draw)
    assert m.sample(PROMPTS, 3, seed=1) == want
    assert torch.equal(between[0], alone)
    assert sorted(m.cache.free) == sorted(free) and not m.cache.lengths_host.any()


def test_a_thread_beside_a_sample(cuda_lib):
    """One thread draws while another scores texts: both as alone."""
    m = model(cache_bits=8)
    text = list(range(300, 390))
    want, alone = m.sample(PROMPTS, 20, seed=2), m.score(3, text)
    torch.cuda.synchronize()
    got, errors = [], []

    def scores():
        try:
            for _ in range(20):
                got.append(m.score(3, text))
        except Exception as e:                   # (seen by the test, not lost with the thread)
            errors.append(e)

    other = threading.Thread(target=scores)
    other.start()
    drawn = [m.sample(PROMPTS, 20, seed=2) for _ in range(5)]
    other.join()
    torch.cuda.synchronize()
    assert not errors and all(d == want for d in drawn) and all(torch.equal(g, alone) for g in got) and len(got) == 20


@pytest.mark.parametrize("temperature", (0.0, 0.8))
@pytest.mark.parametrize("new_tokens", (1, 2, 6))
@pytest.mark.parametrize("bits", (8, 16))
def test_logits_that_are_no_numbers(cuda_lib, bits, new_tokens, temperature):
    """A token whose embedding is broken: its sequence has no token to go on with, which is said, and the cache is as before."""
    m = model(cache_bits=bits)
    m.embed, m.lm_head = m.embed.clone(), m.lm_head.roll(11, 0)      # (one that is whole, and says neither a prompt's last token again nor 9 behind it)
    whole, m.embed[9] = m.embed[9].clone(), float("nan")
    with pytest.raises(ValueError, match="sequence 1 at its token 0"):
        m.sample([[1, 2], [3, 9, 4]], new_tokens, temperature=temperature)
    assert len(m.cache.free) == m.cache.pages and not m.cache.lengths_host.any()
    m.embed[9] = whole
    m.sample([[1, 2], [3, 9, 4]], new_tokens, temperature=temperature)
    first = m.sample([[1, 2]], 1, temperature=0.0)[0][0][0]
    assert first not in (1, 2)
    m.embed[first] = float("inf")                # from the second token on
    if new_tokens > 1:
        with pytest.raises(ValueError, match="sequence 0 at its token 1"):
            m.sample([[1, 2]], new_tokens, temperature=0.0)
    assert m.sample([[1, 2]], 1, temperature=0.0)[0] == [[first]]
