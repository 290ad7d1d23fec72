"""ops.paged_attention over pages of 8 bits against the definition in 64 bits."""
import pytest
import torch

from paged8_util import Case8
from paged_util import assert_within
from relax_b200 import _lib, ops

pytestmark = pytest.mark.gpu


def run(case, **kw):
    got = ops.paged_attention(case.q, *case.args(), starts=case.starts, max_query=max(case.new + [1]), **case.scales(), **kw)
    torch.cuda.synchronize()
    assert ops._lib.lib().b200_device_error_flags() == 0
    return got


def check(case, **kw):
    args = dict(kw)
    for name, kind in (("slopes", torch.float32), ("prefix", torch.int32)):
        if kw.get(name) is not None:
            args[name] = torch.tensor(kw[name], dtype=kind, device="cuda")
    got = run(case, **args)
    assert_within(got, case.reference(**kw), str(kw))
    return got


HEADS = ((4, 4), (8, 2), (5, 1), (14, 2), (32, 1))


@pytest.mark.parametrize("dtype", ("fp16", "bf16"))
@pytest.mark.parametrize("dim", (64, 128))
@pytest.mark.parametrize("heads,kv", HEADS)
@pytest.mark.parametrize("page", (16, 64))
def test_one_row_each(cuda_lib, heads, kv, dim, page, dtype):
    past = [0, 1, 14, 15, 16, 17, 31, 100, 257, 700]
    check(Case8([1] * len(past), past, heads, kv, dim, page, dtype, seed=heads + dim, ragged=False))


@pytest.mark.parametrize("dtype", ("fp16", "bf16"))
@pytest.mark.parametrize("dim", (64, 128))
@pytest.mark.parametrize("page", (16, 32, 128))
@pytest.mark.parametrize("heads,kv", ((4, 4), (6, 2), (7, 1)))
def test_ragged_rows(cuda_lib, heads, kv, page, dim, dtype):
    check(Case8([3, 0, 40, 1, 129, 17], [5, 9, 0, 130, 60, 255], heads, kv, dim, page, dtype, seed=page + heads))


@pytest.mark.parametrize("new", (1, 2, 5, 33, 150))
@pytest.mark.parametrize("kw", (dict(window=1), dict(window=20), dict(window=300), dict(window=9, prefix=[0, 3, 40]), dict(causal=False), dict(cap=5.0),
                                dict(cap=30.0, window=50), dict(cap=1e6), dict(slopes=[0.5, 0.25, 1.0, 0.0]), dict(slopes=[0.1] * 4, cap=20.0),
                                dict(scale=0.03), dict(scale=-0.2), dict(scale=0.0)))
def test_masks_caps_and_biases(cuda_lib, new, kw):
    check(Case8([new, 1, new], [40, 0, 260], 4, 2, seed=new), **kw)


@pytest.mark.parametrize("new", (1, 40))
def test_rows_that_see_nothing_are_zeros(cuda_lib, new):
    case = Case8([new, 2], [0, 30], 4, 2, seed=3)
    case.lengths[0] = 0                          # its rows have no positions
    got = run(case)
    assert (got[:new] == 0).all() and torch.isfinite(got).all() and (got[new:] != 0).any()


@pytest.mark.parametrize("new", (1, 30))
@pytest.mark.parametrize("spread", (1.0, 64.0))
def test_scales_of_very_different_sizes(cuda_lib, new, spread):
    """A value's scale is in its weight: the smallest blocks count with all their bits where the large ones have no weight."""
    check(Case8([new], [333], 4, 1, seed=5, spread=spread), scale=0.02)


def test_small_values_behind_a_large_one(cuda_lib):
    """The first block's values are 2^16 times as large, and nothing looks at them."""
    case = Case8([1], [200], 4, 1, seed=6, spread=1.0)
    page = case.table[0, 0].long()
    case.v_scales[page] = 2.0 ** 5
    case.values[0][:, :16] = case.v8[page].double().cpu() * 2.0 ** 5
    for p in case.table[0, 1:13].long():
        case.v_scales[p] = 2.0 ** -11
    case.values[0][:, 16:] = torch.cat([case.v8[p].double().cpu() for p in case.table[0, 1:13].long()], dim=1)[:, :185] * 2.0 ** -11
    check(case, window=150)
    check(case, slopes=[8.0] * 4)                # no mask: the distance alone hides it


@pytest.mark.parametrize("new", (1, 3, 64))
def test_one_long_sequence_is_cut(cuda_lib, new):
    check(Case8([new], [9000], 4, 1, page=64, seed=7), window=0)


def test_many_sequences(cuda_lib):
    past = [(37 * i) % 300 for i in range(150)]
    check(Case8([1] * 150, past, 8, 2, page=32, seed=8, ragged=False))


@pytest.mark.parametrize("new", (1, 50))
def test_a_page_stride_a_row_stride_and_a_table_of_a_larger_one(cuda_lib, new):
    case = Case8([new, 1], [70, 33], 6, 2, dim=64, seed=9)
    want = run(case)
    pool, kv, page, dim = case.k8.shape
    flat = torch.full((pool, 3 * kv * page * dim + 16), 0x7f, dtype=torch.uint8, device="cuda")
    views = []
    for i, t in enumerate((case.k8, case.v8)):
        v = flat[:, (i + 1) * kv * page * dim: (i + 2) * kv * page * dim].view(pool, kv, page, dim)
        v.copy_(t.view(torch.uint8))
        views.append(v.view(torch.float8_e4m3fn))
    wide = torch.zeros((case.tokens, 9, dim), dtype=case.q.dtype, device="cuda")
    wide[:, 2:8] = case.q
    got = ops.paged_attention(wide[:, 2:8], *views, case.table, case.lengths, starts=case.starts, **case.scales())
    assert torch.equal(got, want)


@pytest.mark.parametrize("new", (1, 40))
def test_streams_and_graphs(cuda_lib, new):
    case = Case8([new, 1, new], [300, 20, 0], 8, 2, seed=10)
    want = run(case)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run(case)
    assert torch.equal(other, want)
    graph, scratch = torch.cuda.CUDAGraph(), ops.paged_attention_scratch("cuda")
    with torch.cuda.graph(graph):
        held = ops.paged_attention(case.q, *case.args(), starts=case.starts, max_query=new, scratch=scratch, **case.scales())
    for _ in range(3):
        held.zero_()
        graph.replay()
        assert torch.equal(held, want)


def test_refusals(cuda_lib):
    case = Case8([1, 1], [20, 30], 4, 2, seed=11, ragged=False)
    good = dict(q=case.q, k_pages=case.k8, v_pages=case.v8, page_table=case.table, lengths=case.lengths, **case.scales())
    ops.paged_attention(**good)
    for bad in (dict(k_scales=None), dict(v_scales=None), dict(k_scales=None, v_scales=None), dict(k_scales=case.k_scales.float()),
                dict(v_scales=case.v_scales[:1]), dict(k_pages=case.k), dict(k_pages=case.k, v_pages=case.v), dict(q=case.q.float()),
                dict(k_scales=case.k_scales.cpu()), dict(k_scales=case.k_scales.transpose(1, 2)), dict(k_pages=case.k8.view(torch.uint8)),
                dict(k_pages=case.k8.view(torch.uint8).view(torch.float8_e5m2))):
        with pytest.raises(ValueError):
            ops.paged_attention(**{**good, **bad})
    with pytest.raises(_lib.B200Error):          # page strides of 8-bit pages are multiples of 16
        flat = torch.zeros((3, 2 * 16 * 128 + 8), dtype=torch.uint8, device="cuda")
        pages = flat[:, : 2 * 16 * 128].view(3, 2, 16, 128).view(torch.float8_e4m3fn)
        ops.paged_attention(**{**good, "k_pages": pages, "v_pages": pages, "k_scales": case.k_scales[:3].contiguous(), "v_scales": case.k_scales[:3].contiguous()})


def test_pages_behind_two_billion_codes(cuda_lib):
    """Append and attention in the last pages of a pool of 2.2e9 codes: the same bits as in a pool of their own."""
    kv, page, dim, pages, used = 8, 128, 128, 17000, 3
    g = torch.Generator(device="cuda").manual_seed(12)
    qkv = torch.randn((300, (16 + 2 * kv) * dim), device="cuda", generator=g).half()
    angle = torch.rand((400, dim // 2), device="cuda", generator=g)
    lengths, starts = torch.tensor([300], dtype=torch.int32, device="cuda"), torch.tensor([0, 300], dtype=torch.int32, device="cuda")
    got = []
    for pool in (used, pages):
        k, v = (torch.zeros((pool, kv, page, dim), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in "kv")
        scales = {n: torch.ones((pool, kv, page // 16), dtype=torch.float16, device="cuda") for n in ("k_scales", "v_scales")}
        table = torch.arange(pool - used, pool, dtype=torch.int32, device="cuda").flip(0)[None].contiguous()
        q = ops.paged_rope_append(qkv, angle.cos(), angle.sin(), k, v, table, lengths, starts=starts, **scales)
        many = ops.paged_attention(q, k, v, table, lengths, starts=starts, max_query=300, **scales)
        few = ops.paged_attention(q[299:].contiguous(), k, v, table, lengths, **scales)
        got.append((q, many, few, k[-used:].view(torch.uint8).clone(), scales["v_scales"][-used:].clone()))
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_calls_on_two_streams_at_once(cuda_lib):
    """Attention with a scratch of each stream's own beside plans and sampling on the other: what each gives alone."""
    case = Case8([1, 40], [700, 200], 8, 2, seed=13)
    g = torch.Generator(device="cuda").manual_seed(14)
    logits, u = torch.randn((9, 40000), device="cuda", generator=g), torch.rand(9, device="cuda", generator=g)
    want = run(case), ops.sample_tokens(logits, u, top_p=0.9)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for i in range(12):
        with torch.cuda.stream(streams[i % 3]):
            got.append((ops.paged_attention(case.q, *case.args(), starts=case.starts, max_query=40, **case.scales()), ops.sample_tokens(logits, u, top_p=0.9)))
    torch.cuda.synchronize()
    for a, drawn in got:
        assert torch.equal(a, want[0]) and torch.equal(drawn.token, want[1].token) and torch.equal(drawn.logprob, want[1].logprob)
