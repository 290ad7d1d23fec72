"""Places and pages of a call that keeps its tables on the device: nobody else gets them before it returns."""
import copy
import pickle
import threading

import pytest

torch = pytest.importorskip("torch")

from relax_b200 import paged
from test_paged_cache_cpu import decoder


def cache(pages=10):
    return paged.PagedCache(1, 1, 64, 16, pages=pages, batch=4, max_tokens=100, device="cpu")


def test_pages_that_are_held_are_nobody_elses():
    c = cache()
    free = list(c.free)
    pages = c.hold([17, 40])
    assert len(pages) == 5 and sorted(pages + c.free) == sorted(free) and c.free == free[:5]
    c.extend(3, 80)
    assert not set(c.table_host[3, :5].tolist()) & set(pages)
    with pytest.raises(MemoryError):
        c.extend(2, 1)
    c.release(3)
    c.give_back(2, pages)
    assert sorted(c.free) == sorted(free) and not c.lengths_host.any() and not c.held


def test_places_that_are_held_are_in_use():
    c = cache()
    pages = c.hold([1, 1])
    for call in (lambda: c.hold([1]), lambda: c.extend(0, 1), lambda: c.extend(1, 1), lambda: c.shrink(1, 1), lambda: c.release(0)):
        with pytest.raises(ValueError, match="in use"):
            call()
    assert c.length(0) == c.length(1) == 1 and c.length(2) == 0
    c.extend(2, 5)
    c.give_back(2, pages)
    c.extend(0, 1)
    with pytest.raises(ValueError, match="in use"):
        c.hold([0])


def test_what_has_no_room_changes_nothing():
    c = cache(pages=4)
    free = list(c.free)
    with pytest.raises(ValueError, match="100"):
        c.hold([101])
    with pytest.raises(MemoryError):
        c.hold([33, 32])
    with pytest.raises(IndexError):
        c.hold([1] * 5)
    assert c.free == free and not c.lengths_host.any() and not c.held
    assert c.hold([0, 0]) == [] and c.free == free and c.held == {0, 1}


def test_a_call_that_fails_gives_back_what_it_held():
    m = decoder()
    free = list(m.cache.free)
    with pytest.raises(Exception):               # there is no GPU here, or none for this decoder's tensors
        m.sample([[1, 2], [3]], 5)
    assert m.cache.free == free and not m.cache.lengths_host.any() and not m.cache.held
    with pytest.raises(Exception):
        m.sample([[1, 2], [3]], 5, uniform=torch.zeros((5, 2)))
    assert m.cache.free == free and not m.cache.held


def test_threads_share_the_pool():
    """Eight threads that take and give back at once: no page is ever two threads'."""
    c = paged.PagedCache(1, 1, 64, 16, pages=64, batch=9, max_tokens=100, device="cpu")
    taken, wrong = [set() for _ in range(9)], []

    def holds():
        for _ in range(300):
            taken[0] = set(pages := c.hold([90]))
            if any(taken[0] & t for t in taken[1:]):
                wrong.append(0)
            taken[0] = set()
            c.give_back(1, pages)

    def extends(i):
        for n in range(300):
            c.extend(i, 1 + n % 100)
            taken[i] = set(c.table_host[i, : -(-c.length(i) // 16)].tolist())
            if any(taken[i] & t for j, t in enumerate(taken) if j != i):
                wrong.append(i)
            taken[i] = set()
            c.release(i)

    threads = [threading.Thread(target=holds)] + [threading.Thread(target=extends, args=(i,)) for i in range(1, 9)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and sorted(c.free) == list(range(64)) and not c.lengths_host.any()


@pytest.mark.parametrize("again", (copy.deepcopy, lambda c: pickle.loads(pickle.dumps(c))))
def test_a_cache_is_copied_with_what_it_holds(again):
    c = cache()
    c.extend(3, 30)
    pages = c.hold([17])
    other = again(c)
    assert other.free == c.free and other.held == {0} and (other.table_host == c.table_host).all()
    other.give_back(1, pages)
    assert c.held == {0} and c.length(0) == 17 and other.length(0) == 0 and len(other.free) == len(c.free) + 2
