"""What the operators over 8-bit pages, the plan and sampling refuse without a GPU, and the host side of the cache in 8 bits."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from relax_b200 import _lib, ops, paged


def test_a_cache_in_eight_bits_has_scales():
    c = paged.PagedCache(layers=2, kv_heads=3, head_dim=64, page_size=32, pages=5, batch=2, max_tokens=64, dtype=torch.float8_e4m3fn, device="cpu")
    assert c.k[1].dtype is torch.float8_e4m3fn and sorted(c.scales[0]) == ["k_scales", "v_scales"]
    assert c.scales[1]["v_scales"].shape == (5, 3, 2) and c.scales[1]["v_scales"].dtype is torch.float16
    assert paged.PagedCache(layers=2, kv_heads=3, head_dim=64, page_size=32, pages=5, batch=2, max_tokens=64, device="cpu").scales == [{}, {}]


def test_cpu_tensors_are_refused():
    k = torch.zeros((3, 1, 16, 64), dtype=torch.float8_e4m3fn)
    scales = dict(k_scales=torch.ones((3, 1, 1), dtype=torch.float16), v_scales=torch.ones((3, 1, 1), dtype=torch.float16))
    i32 = dict(dtype=torch.int32)
    table, lengths = torch.zeros((1, 2), **i32), torch.ones(1, **i32)
    q = torch.zeros((1, 2, 64), dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_attention(q, k, k, table, lengths, **scales)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_rope_append(torch.zeros((1, 4 * 64), dtype=torch.float16), torch.zeros((4, 32)), torch.zeros((4, 32)), k, k, table, lengths, **scales)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_plan(table, lengths, lengths, lengths, lengths, 16, 4)
    with pytest.raises(ValueError, match="CUDA"):
        ops.sample_tokens(torch.zeros((1, 9)), torch.zeros(1))


@pytest.mark.parametrize("change", (dict(k_scales=None), dict(v_scales=None), dict(k_scales=None, v_scales=None), dict(k_scales=torch.ones((3, 1, 1))),
                                    dict(v_scales=torch.ones((3, 1, 2), dtype=torch.float16)), dict(q=torch.zeros((1, 2, 64)))))
def test_scales_that_do_not_fit(change):
    k = torch.zeros((3, 1, 16, 64), dtype=torch.float8_e4m3fn)
    good = dict(q=torch.zeros((1, 2, 64), dtype=torch.float16), k_scales=torch.ones((3, 1, 1), dtype=torch.float16), v_scales=torch.ones((3, 1, 1), dtype=torch.float16))
    with pytest.raises(ValueError, match="scales|rows"):
        ops.paged_attention(k_pages=k, v_pages=k, page_table=torch.zeros((1, 2), dtype=torch.int32), lengths=torch.ones(1, dtype=torch.int32), **{**good, **change})


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU behaviour")
def test_the_c_entries_fail_loudly_without_a_gpu():
    L = _lib.lib()
    p = torch.zeros(4096, dtype=torch.int32).data_ptr()
    c = _lib.PagedCache(_lib.F16, 1, 64, 16, 3, 1024, 1024, p, p, 1, 2, 1, 2, 1, p, p, None)
    s, a = _lib.PagedScales(p, p), _lib.PagedAttention(p, 128, p, 2, 1, 0, 1.0, 0.0, None, None)
    attention = lambda s=s: L.b200_paged8_attention(ctypes.byref(c), ctypes.byref(s) if s else None, ctypes.byref(a), p, 4096, None)  # noqa: E731
    append = lambda s=s: L.b200_paged8_rope_append(ctypes.byref(c), ctypes.byref(s) if s else None, p, 256, 2, p, p, 4, 64, 0, None, p, None)  # noqa: E731
    assert attention() == append() == _lib.ENODEVICE
    assert attention(None) == append(None) == _lib.EINVAL and "scales" in _lib.last_error()
    assert attention(_lib.PagedScales(p, None)) == append(_lib.PagedScales(p + 1, p)) == _lib.EINVAL
    c.k_page_stride = 1032
    assert attention() == append() == _lib.EINVAL and "multiples of 16" in _lib.last_error()

    plan = dict(batch=1, table_width=2, page_size=16, max_tokens=0, table_stride=2, pages=5, rows=4, page_table=p, lengths=p, counts=p, free_pages=p, free_count=p,
                lengths_out=p, starts=p, positions=p, slots=p, free_count_out=p, status=p)
    call = lambda **kw: L.b200_paged_plan(ctypes.byref(_lib.PagedPlan(**{**plan, **kw})), None)  # noqa: E731
    assert call() == _lib.ENODEVICE and L.b200_paged_plan(None, None) == _lib.EINVAL
    for bad in (dict(page_size=24), dict(batch=-1), dict(batch=8193), dict(table_width=0), dict(batch=2, table_stride=1), dict(pages=0), dict(rows=-1), dict(rows=1 << 27),
                dict(max_tokens=-1), dict(table_width=1 << 30), *({n: None} for n in ("page_table", "lengths", "counts", "free_pages", "free_count", "lengths_out",
                                                                                      "starts", "positions", "slots", "free_count_out", "status"))):
        assert call(**bad) == _lib.EINVAL, bad

    how = _lib.Sampling(1.0, 1.0, 0.0, 0, None, None, None, None)
    draw = lambda logits=p, dtype=_lib.F32, stride=9, uniform=p, how=ctypes.byref(how), token=p, rows=1, V=9: L.b200_sample_tokens(  # noqa: E731
        logits, dtype, stride, uniform, how, token, None, rows, V, None)
    assert draw() == _lib.ENODEVICE and draw(rows=0) == _lib.OK
    for bad in (dict(logits=None), dict(logits=p + 2), dict(dtype=7), dict(stride=8, rows=2), dict(uniform=None), dict(how=None), dict(token=None), dict(rows=-1),
                dict(V=0), dict(V=(1 << 31) - 65536)):
        assert draw(**bad) == _lib.EINVAL, bad
