"""Attention over the paged cache against its definition in 64 bits: lengths around the units and pages, head groups, masks that leave
rows empty, garbage where nobody may look, strides, streams, and what is refused."""
import pytest

torch = pytest.importorskip("torch")

from paged_util import Case, assert_within
from relax_b200 import B200Error, _lib, ops

pytestmark = pytest.mark.gpu


def run(c, **kw):
    prefix = kw.pop("prefix", None)
    slopes = kw.pop("slopes", None)
    out = torch.full((c.tokens, c.heads, c.dim), float("nan"), dtype=c.q.dtype, device="cuda")
    ops.paged_attention(c.q, *c.args(), starts=c.starts, max_query=max(c.new), out=out,
                        prefix=None if prefix is None else torch.tensor(prefix, dtype=torch.int32).cuda(),
                        slopes=None if slopes is None else torch.tensor(slopes, dtype=torch.float32).cuda(), **kw)
    torch.cuda.synchronize()
    assert_within(out, c.reference(prefix=prefix, slopes=slopes, **kw))
    return out


# one token each: lengths around the unit of 16, the page, the chunk; an empty and a one-token sequence among them
LENGTHS = [1, 2, 15, 16, 17, 31, 33, 64, 65, 127, 129, 300, 1000, 2049]


@pytest.mark.parametrize("heads,kv", [(4, 4), (8, 2), (10, 2), (8, 1), (24, 2), (16, 1)])
@pytest.mark.parametrize("dim,page,dtype", [(128, 16, "fp16"), (64, 32, "fp16"), (128, 128, "bf16"), (64, 16, "bf16")])
def test_one_token_each(cuda_lib, heads, kv, dim, page, dtype):
    run(Case([1] * len(LENGTHS), [n - 1 for n in LENGTHS], heads, kv, dim, page, dtype, ragged=False))


@pytest.mark.parametrize("length", [1, 17, 700, 5000])
def test_one_sequence_alone(cuda_lib, length):
    run(Case([1], [length - 1], 8, 8, ragged=False))
    run(Case([1], [length - 1], 8, 1, ragged=True))


# ragged rows: prompts, chunks behind a context, sequences without rows, a row group that is no power of two
RAGGED = [([5, 1, 130, 0, 17], [0, 40, 0, 9, 300]), ([1, 2, 3, 4], [0, 0, 15, 16]), ([64, 65], [64, 1]), ([257], [0]), ([33], [1000])]


@pytest.mark.parametrize("new,past", RAGGED)
@pytest.mark.parametrize("heads,kv,dim,page,dtype", [(4, 4, 128, 16, "fp16"), (6, 2, 64, 32, "bf16"), (8, 1, 128, 64, "fp16"), (14, 2, 128, 128, "bf16"),
                                                     (32, 1, 64, 16, "fp16"), (100, 1, 128, 16, "fp16")])
def test_ragged(cuda_lib, new, past, heads, kv, dim, page, dtype):
    run(Case(new, past, heads, kv, dim, page, dtype, stride=64))


MASKS = [dict(window=1), dict(window=16), dict(window=100), dict(cap=5.0), dict(cap=30.0, window=77), dict(causal=False), dict(scale=0.3)]


@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("new,past", [([1, 1, 1], [0, 50, 700]), ([3, 40, 1], [0, 200, 31]), ([150, 1, 300], [7, 0, 0])])
@pytest.mark.parametrize("dim,dtype", [(128, "fp16"), (64, "bf16")])
def test_masks_and_caps(cuda_lib, mask, new, past, dim, dtype):
    c = Case(new, past, 8, 2, dim, 32, dtype)
    run(c, **mask)
    if mask.get("causal", True):
        run(c, prefix=[0, 5, 1000], **mask)
        run(c, prefix=[70, 300, 33], **mask)
    run(c, slopes=[2.0 ** -i for i in range(8)], **mask)


def test_rows_without_a_place_are_zero(cuda_lib):
    """More rows than the sequence has tokens: the first ones lie before its beginning; and an empty sequence."""
    c = Case([5, 2, 3], [-3, -2, -9], 4, 2)
    out = run(c)
    assert (out[:3] == 0).all() and (out[3:5] != 0).any() and (out[5:] == 0).all()
    out = run(c, causal=False)
    assert (out[:3] == 0).all() and (out[5:] == 0).all()
    run(c, prefix=[1, 1, 1])


def test_what_nobody_sees_may_be_anything(cuda_lib):
    """Tokens behind the window hold infinities and NaN (their pages belong to others by now), keys and values; so does the space
    behind the last token (NaN everywhere in these cases)."""
    for new in ([1], [40], [200]):
        c = Case(new, [333], 8, 2, ragged=True)
        oldest = 333 - 64 + 1                             # the first row's window begins here
        for b, page in enumerate(c.table[0, : -(-c.length[0] // 16)].tolist()):
            rows = slice(0, max(0, min(16, oldest - 16 * b)))
            if b * 16 >= 5:
                c.k[page, :, rows] = float("inf")
                c.v[page, :, rows] = float("nan")
        run(c, window=64)
        for page in (c.table[0, 0].item(),):              # four tokens at the front stay visible, those behind them do not
            c.v[page, :, 4:16] = float("nan")
            c.k[page, :, 4:16] = float("nan")
        run(c, window=64, prefix=[4])


def test_lowest_scores_and_large_ones(cuda_lib):
    """Scores near fp32's end, all equal, and far apart."""
    c = Case([1, 30], [90, 0], 4, 2)
    c.q.mul_(60.0)
    run(c)
    run(c, scale=-2.0)
    c.q.zero_()
    run(c)


def test_long_cache(cuda_lib):
    """Positions past 2^31 elements of the pool: a page far behind the others."""
    kv, page, dim = 8, 128, 128
    pool = 2 ** 31 // (kv * page * dim) + 40
    k = torch.zeros((pool, kv, page, dim), dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    for pages in ([pool - 1, 3, pool - 7], [2, pool - 2]):
        c = Case([1 if len(pages) == 2 else 150], [page * (len(pages) - 1) + 9 if len(pages) == 2 else 200], 16, kv, dim, page)
        own = -(-c.length[0] // page)
        for i in range(own):
            k[pages[i]], v[pages[i]] = c.k[c.table[0, i]], c.v[c.table[0, i]]
        c.k, c.v = k, v
        c.table = torch.tensor([pages], dtype=torch.int32).cuda()
        run(c)


def test_views_streams_and_graphs(cuda_lib):
    c = Case([1] * 5, [30, 600, 2, 1000, 77], 16, 4, ragged=False)
    want = run(c)
    qkv = torch.randn((5, (16 + 8) * 128), dtype=torch.float16, device="cuda")
    qkv[:, : 16 * 128] = c.q.view(5, -1)
    table = torch.full((5, 2 * c.table.shape[1]), 7, dtype=torch.int32, device="cuda")
    table[:, : c.table.shape[1]] = c.table
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.paged_attention(qkv[:, : 16 * 128].view(5, 16, 128), c.k, c.v, table[:, : c.table.shape[1]], c.lengths)
    side.synchronize()
    assert torch.equal(got, want)
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(want)
    with torch.cuda.graph(graph):
        ops.paged_attention(c.q, *c.args(), out=out)
        ops.paged_attention(c.q, *c.args(), out=out)
    for _ in range(3):
        out.fill_(float("nan"))
        graph.replay()
        again = ops.paged_attention(c.q, *c.args())
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(again, want)


def test_the_same_bits_every_time(cuda_lib):
    for c in (Case([1] * 3, [5000, 3, 900], 8, 2, ragged=False), Case([700, 20], [0, 3000], 8, 2)):
        first = run(c)
        for _ in range(20):
            assert torch.equal(run_again(c), first)


def run_again(c):
    out = ops.paged_attention(c.q, *c.args(), starts=c.starts, max_query=max(c.new))
    torch.cuda.synchronize()
    return out


def test_many_sequences(cuda_lib):
    """More sequences than the scheduling warp keeps in shared memory, some without rows, one much longer than the others."""
    new = [(i * 37) % 50 for i in range(90)]
    past = [(i * 53) % 200 for i in range(90)]
    new[40], past[40] = 300, 3000
    run(Case(new, past, 4, 2, 64, 32))
    run(Case([1] * 150, [(i * 97) % 700 for i in range(150)], 4, 1, 128, 16, ragged=False))


@pytest.mark.parametrize("new,past", [(40, 20000), (513, 5000), (17, 9000)])
def test_a_part_of_a_long_text(cuda_lib, new, past):
    """Few rows behind a long context: the context is cut into chunks that several CTAs share."""
    c = Case([new], [past], 8, 2, 128, 128)
    first = run(c)
    assert torch.equal(run_again(c), first)
    run(c, window=2000, prefix=[700])
    run(c, cap=7.0)
    run(c, slopes=[2.0 ** -(i + 4) for i in range(8)])


@pytest.mark.parametrize("heads,kv,dim,dtype", [(14, 2, 128, "bf16"), (8, 2, 64, "fp16"), (4, 4, 128, "fp16")])
@pytest.mark.parametrize("new,past", [([100], [3000]), ([70, 1, 40], [2500, 5, 4000]), ([300], [900])])
def test_parts_that_are_joined(cuda_lib, new, past, heads, kv, dim, dtype):
    """Many rows of a long text on few key heads: cut into parts, some of which a mask leaves empty, with tiles that are not full."""
    c = Case(new, past, heads, kv, dim, 64, dtype)
    run(c)
    run(c, cap=5.0)
    run(c, cap=200.0, window=500, prefix=[300] * len(new))
    run(c, slopes=[2.0 ** -i for i in range(heads)], causal=False)


def test_rows_by_a_bound_only(cuda_lib):
    """max_query is a bound: a larger one, or none, gives the same values by another kernel."""
    c = Case([3, 1, 4], [100, 30, 0], 4, 2)
    want = run(c)
    for most in (4, 5, 100, None):
        out = ops.paged_attention(c.q, *c.args(), starts=c.starts, max_query=most)
        torch.cuda.synchronize()
        assert_within(out, c.reference())
        assert (out - want).abs().max() < 2e-3


def test_the_way_without_the_extension(cuda_lib, monkeypatch):
    c = Case([5, 60], [100, 3], 8, 2)
    want = run(c, window=50)
    monkeypatch.setattr(ops, "_native", False)
    monkeypatch.setattr(ops, "_torch_call", lambda: False)
    assert torch.equal(run(c, window=50), want)


def test_a_prompt_in_a_graph(cuda_lib):
    c = Case([200, 40], [0, 900], 8, 2)
    want = run(c)
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(want)
    with torch.cuda.graph(graph):
        ops.paged_attention(c.q, *c.args(), starts=c.starts, max_query=200, out=out)
    for _ in range(3):
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert cuda_lib.b200_device_error_flags() == 0


def test_refusals(cuda_lib):
    c = Case([1, 1], [3, 4], 8, 2, ragged=False)

    def call(q=c.q, k=c.k, v=c.v, table=c.table, lengths=c.lengths, **kw):
        return ops.paged_attention(q, k, v, table, lengths, **kw)

    call()
    for bad in (dict(q=c.q.float()), dict(q=c.q[:, :, :64]), dict(q=c.q[:, :7]), dict(k=c.k[:, :, :8].contiguous(), v=c.v[:, :, :8].contiguous()),
                dict(k=c.k.transpose(1, 2)), dict(v=c.v.bfloat16()), dict(table=c.table.long()), dict(table=c.table.t()),
                dict(lengths=c.lengths.long()), dict(lengths=c.lengths[:1]), dict(q=c.q[:1]), dict(starts=torch.zeros(2, dtype=torch.int32).cuda()),
                dict(window=-1), dict(window=3, causal=False), dict(cap=-1.0), dict(cap=float("nan")), dict(scale=float("nan")),
                dict(slopes=torch.zeros(7).cuda()), dict(prefix=torch.zeros(3, dtype=torch.int32).cuda()), dict(out=c.q[:1]),
                dict(lengths=c.lengths.cpu()), dict(scratch=torch.zeros(16, dtype=torch.uint8).cuda()), dict(q=c.q.cpu())):
        with pytest.raises((ValueError, B200Error)):
            call(**bad)
    assert ops.paged_attention(c.q[:0], c.k, c.v, c.table[:0], c.lengths[:0]).shape == (0, 8, 128)


def test_the_c_entry_refuses(cuda_lib):
    import ctypes

    c = Case([1, 1], [3, 4], 8, 2, ragged=False)
    cache = ops._paged_cache(c.q, *c.args(), None, None)
    args = _lib.PagedAttention(c.q.data_ptr(), 1024, c.q.data_ptr(), 8, 1, 0, 1.0, 0.0, None, None)
    scratch = ops.paged_attention_scratch("cuda")

    def call(cache=cache, args=args, scratch=scratch.data_ptr(), size=scratch.numel()):
        return cuda_lib.b200_paged_attention(cache and ctypes.byref(cache), args and ctypes.byref(args), scratch, size, 0)

    def but(struct, **kw):
        copy = type(struct)()
        ctypes.memmove(ctypes.byref(copy), ctypes.byref(struct), ctypes.sizeof(struct))
        for name, value in kw.items():
            setattr(copy, name, value)
        return copy

    for kw in (dict(cache=None), dict(args=None), dict(scratch=None), dict(size=100)):
        assert call(**kw) == _lib.EINVAL, kw
    for name, value in (("dtype", 2), ("head_dim", 96), ("page_size", 48), ("page_size", 8), ("kv_heads", 0), ("batch", -1), ("tokens", 1), ("pages", 0),
                        ("table_width", 0), ("k_page_stride", 100), ("v_page_stride", 8), ("k_pages", None), ("v_pages", c.v.data_ptr() + 8),
                        ("page_table", None), ("lengths", None), ("table_stride", 0), ("table_width", 2 ** 28)):
        assert call(cache=but(cache, **{name: value})) == _lib.EINVAL, name
    for name, value in (("q", None), ("q", c.q.data_ptr() + 2), ("q_stride", 1000), ("q_stride", 1028), ("out", None), ("heads", 7), ("heads", 0),
                        ("heads", 2 * 129), ("window", -1), ("scale", float("nan")), ("cap", -1.0)):
        assert call(args=but(args, **{name: value})) == _lib.EINVAL, name
