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
