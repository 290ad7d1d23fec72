"""Host logic of the paged cache, the rotary tables, and what the operators refuse without a GPU."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from relax_b200 import _lib, decoder, ops, paged


def cache(**kw):
    return paged.PagedCache(**{**dict(layers=1, kv_heads=1, head_dim=64, page_size=16, pages=6, batch=3, max_tokens=64, device="cpu"), **kw})


def test_pages_are_handed_out_and_given_back():
    c = cache()
    c.extend(0, 17)
    c.extend(1, 16)
    c.extend(1, 1)
    assert c.lengths_host.tolist() == [17, 17, 0] and len(c.free) == 2
    used = c.table_host[:2, :2].ravel().tolist()
    assert len(set(used)) == 4 and (c.table_host[:2, 2:] == -1).all()
    table, lengths = c.tables([1, 0])
    assert table.shape == (2, 2) and table.dtype == torch.int32 and lengths.tolist() == [17, 17] and table[0].tolist() == used[2:]
    with pytest.raises(MemoryError):
        c.extend(2, 33)
    with pytest.raises(ValueError):
        c.extend(2, 65)
    with pytest.raises(ValueError):
        c.extend(2, -1)
    assert c.lengths_host.tolist() == [17, 17, 0] and len(c.free) == 2 and (c.table_host[2] == -1).all()
    c.extend(0, 20)
    c.shrink(0, 20)
    assert c.lengths_host.tolist() == [17, 17, 0] and len(c.free) == 2 and (c.table_host[0, 2:] == -1).all()
    with pytest.raises(ValueError):
        c.shrink(0, 18)
    c.release(0)
    c.extend(2, 64)
    assert len(c.free) == 0
    c.release(1)
    c.release(2)
    assert sorted(c.free) == list(range(6)) and (c.table_host == -1).all() and c.tables([0])[0].shape == (1, 1)


def test_tables_and_their_scalings():
    cos, sin = paged.rope_tables(50, 128, device="cpu")
    want = decoder.rope_tables(50, 128, 10000.0, "cpu")
    assert torch.equal(cos, want[0]) and torch.equal(sin, want[1])
    angle = lambda **kw: torch.atan2(*paged.rope_tables(2, 32, device="cpu", **kw)[::-1])[1].double()      # of position 1
    plain = angle()
    assert torch.allclose(angle(scaling=dict(kind="linear", factor=4.0)), plain / 4, rtol=1e-6)
    base = angle(scaling=dict(kind="base", factor=8.0))
    assert torch.isclose(base[0], plain[0]) and torch.isclose(base[-1], plain[-1] / 8, rtol=1e-6) and (base <= plain).all()
    parts = angle(scaling=dict(kind="parts", factor=8.0, original=2000, low=1.0, high=4.0))
    turns = 2000 * plain / (2 * np.pi)
    assert torch.allclose(parts[turns >= 4], plain[turns >= 4]) and torch.allclose(parts[turns <= 1], plain[turns <= 1] / 8, rtol=1e-6)
    between = (turns > 1) & (turns < 4)
    assert between.any() and ((parts < plain) & (parts > plain / 8))[between].all()
    louder = paged.rope_tables(9, 32, device="cpu", scaling=dict(kind="linear", factor=2.0, magnitude=1.25))
    assert torch.allclose(louder[0] ** 2 + louder[1] ** 2, torch.tensor(1.25 ** 2))
    for bad in (dict(kind="other"), dict(kind="linear", factor=2.0, more=1), dict(kind="parts", factor=2.0, original=9, low=3.0, high=2.0)):
        with pytest.raises(ValueError):
            paged.rope_tables(4, 32, scaling=bad, device="cpu")
    with pytest.raises(ValueError):
        paged.PagedConfig(heads=6, kv_heads=4)


def test_cpu_tensors_are_refused():
    k = torch.zeros((3, 1, 16, 64), dtype=torch.float16)
    table, lengths = torch.zeros((1, 2), dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q = torch.zeros((1, 2, 64), dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_attention(q, k, k, table, lengths)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_rope_append(torch.zeros((1, 4 * 64), dtype=torch.float16), torch.zeros((4, 32)), torch.zeros((4, 32)), k, k, table, lengths)
    with pytest.raises(ValueError, match="CUDA"):
        ops.token_logprobs(torch.zeros((1, 9)), torch.zeros(1, dtype=torch.int32))


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU behaviour")
def test_the_c_entries_fail_loudly_without_a_gpu():
    import ctypes

    L = _lib.lib()
    buffer = torch.zeros(4096, dtype=torch.int32)
    p = buffer.data_ptr()
    c = _lib.PagedCache(_lib.F16, 1, 64, 16, 3, 1024, 1024, p, p, 1, 2, 1, 2, 1, p, p, None)
    a = _lib.PagedAttention(p, 128, p, 2, 1, 0, 1.0, 0.0, None, None)
    assert L.b200_paged_attention(ctypes.byref(c), ctypes.byref(a), p, 4096, None) == _lib.ENODEVICE
    assert L.b200_paged_rope_append(ctypes.byref(c), p, 256, 2, p, p, 4, 64, 0, None, p, None) == _lib.ENODEVICE
    assert L.b200_token_logprobs(p, _lib.F32, 9, p, p, p, None, None, 1, 9, 0, None) == _lib.ENODEVICE
    assert L.b200_paged_attention_scratch_bytes() == -1
    c.page_size = 17
    assert L.b200_paged_attention(ctypes.byref(c), ctypes.byref(a), p, 4096, None) == _lib.EINVAL and "page_size" in _lib.last_error()
