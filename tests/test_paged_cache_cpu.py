"""What the paged cache and its decoder refuse, and what they leave behind them then, without a GPU."""
import pytest

torch = pytest.importorskip("torch")

from relax_b200 import paged


@pytest.mark.parametrize("page_size", [16, 128])
def test_a_sequence_holds_max_tokens_and_no_more(page_size):
    """The rest of the last page is no room: the rotary tables end at max_tokens."""
    c = paged.PagedCache(1, 1, 64, page_size, pages=20, batch=2, max_tokens=100, device="cpu")
    with pytest.raises(ValueError, match="100"):
        c.extend(0, 101)
    c.extend(0, 100)
    for more in (1, 12, 28):
        with pytest.raises(ValueError, match="100"):
            c.extend(0, more)
    c.extend(0, 0)
    c.extend(1, 99)
    c.extend(1, 1)
    with pytest.raises(ValueError, match="100"):
        c.extend(1, 1)
    assert c.lengths_host.tolist() == [100, 100] and len(c.free) == 20 - 2 * -(-100 // page_size)


def decoder(**kw):
    """A decoder whose first operator fails: there is no GPU here."""
    cfg = paged.PagedConfig(hidden=128, heads=2, kv_heads=1, inter=128, layers=1, vocab=50, head_dim=64, rotary=64, **kw)
    embed = torch.zeros((50, 128), dtype=torch.float16)
    return paged.PagedDecoder(cfg, [], embed, torch.ones(128, dtype=torch.float16), embed, batch=3, max_tokens=40, device="cpu")


def test_a_call_that_fails_leaves_the_sequences_as_they_were():
    m = decoder()
    m.cache.extend(1, 17)
    table, free = m.cache.table_host.copy(), list(m.cache.free)

    def as_it_was():
        return m.cache.lengths_host.tolist() == [0, 17, 0] and (m.cache.table_host == table).all() and sorted(m.cache.free) == sorted(free)

    for tokens in ([[1, 2], ["a", 3]], [[1, 2], [None]], [[1, 2], [3.5]]):
        with pytest.raises(TypeError):
            m.forward([0, 1], tokens)
        assert as_it_was(), tokens
    for tokens in ([[1, 2], [50]], [[-1], [3]], [[1], [2 ** 40]]):
        with pytest.raises(ValueError, match="0 to 49"):
            m.forward([0, 1], tokens)
        assert as_it_was(), tokens
    with pytest.raises(Exception):                  # behind the tables: the first operator finds no GPU
        m.forward([0, 1], [[1, 2], [3]])
    assert as_it_was()
    for error in (MemoryError, KeyboardInterrupt):
        def fails(*args, error=error):
            raise error
        m._forward = fails
        with pytest.raises(error):
            m.forward([2, 1], [[1, 2] * 17, [3]])
        assert as_it_was()


def test_a_negative_number_names_no_place():
    """-1 would be another name of the last place: the same sequence twice in a call, and a text scored in a place that is in use."""
    m = decoder()
    m.cache.extend(2, 5)
    for call in (lambda: m.forward([-1, 2], [[1], [2]]), lambda: m.forward([3], [[1]]), lambda: m.score(-1, [1, 2]),
                 lambda: m.cache.extend(-1, 1), lambda: m.cache.shrink(-1, 1), lambda: m.cache.release(-1), lambda: m.cache.release(3)):
        with pytest.raises(IndexError, match="place"):
            call()
        assert m.cache.lengths_host.tolist() == [0, 0, 5] and len(m.cache.free) == m.cache.pages - 1


def test_no_tokens_asked_for():
    """A list for every sequence all the same, and nothing left in the cache."""
    m = decoder()
    for more in (dict(), dict(top=5)):
        assert m.generate([[1, 2], [3]], 0, **more) == ([[], []], [[], []], [[], []])
    assert m.cache.lengths_host.tolist() == [0, 0, 0]
