"""What the tokens that are left of a block of 16 hold in 8 bits when others have come and gone, by a call that failed or by shrink()."""
import pytest

torch = pytest.importorskip("torch")

from relax_b200 import ops
from test_paged_decoder_gpu import model

pytestmark = pytest.mark.gpu


def held(m, seq, n):
    """(values, scales) of the first n tokens of a sequence, each [layers, 2, n, kv, dim] in 64 bits."""
    page = m.cfg.page_size
    at = [(int(m.cache.table_host[seq, t // page]), t % page) for t in range(n)]
    codes = [[torch.stack([p[i, :, o].double() for i, o in at]) for p in kv] for kv in zip(m.cache.k, m.cache.v)]
    scales = [[torch.stack([s[n][i, :, o // 16].double()[:, None] for i, o in at]) for n in ("k_scales", "v_scales")] for s in m.cache.scales]
    scales = torch.stack([torch.stack(x) for x in scales])
    return torch.stack([torch.stack(x) for x in codes]) * scales, scales


def loud(m, token, factor=40.0):
    """A token whose values are large in every layer."""
    for w in m.layers:
        w["qkv"] = (w["qkv"][0], w["qkv"][1] * factor)
    m.embed[token] *= 4


@pytest.mark.parametrize("page", (16, 64))
@pytest.mark.parametrize("n", (1, 5, 16, 21))
@pytest.mark.parametrize("way", ("a call that fails", "shrink"))
def test_what_is_left(cuda_lib, monkeypatch, way, n, page):
    m = model(cache_bits=8, page_size=page)
    m.embed = m.embed.clone()
    m.forward([0, 1], [list(range(10, 10 + n)), [4] * 20])
    before, was = held(m, 0, n)
    table, free = m.cache.table_host.copy(), list(m.cache.free)
    loud(m, 7)
    if way == "shrink":
        m.forward([0], [[7, 7]])
        m.cache.shrink(0, 2)
    else:
        attention, calls = ops.paged_attention, []

        def fails(*args, **kw):
            calls.append(0)
            if len(calls) == 2:                  # (the second layer's keys are stored)
                raise RuntimeError("no more")
            return attention(*args, **kw)

        monkeypatch.setattr(ops, "paged_attention", fails)
        with pytest.raises(RuntimeError, match="no more"):
            m.forward([0, 1], [[7, 7], [7]])
        monkeypatch.setattr(ops, "paged_attention", attention)
    assert m.cache.length(0) == n and m.cache.length(1) == 20
    assert sorted(m.cache.free) == sorted(free) and (m.cache.table_host == table).all()
    after, now = held(m, 0, n)
    assert (now >= was).all()
    off = (after - before).abs()
    grown = now > was
    assert (off[~grown.expand_as(off)] == 0).all()
    assert (off <= 2.0 ** -10 * now).all() and (off[before.abs() >= 2.0 ** -6 * now] == 0).all()
    whole = n // 16 * 16
    assert (off[:, :, :whole] == 0).all() and not grown[:, :, :whole].any()      # a block that was full is not touched
    if n % 16:
        assert grown[:, :, whole:].any()                                        # (the case is one)
    m.forward([0], [[3]])                        # and it goes on
