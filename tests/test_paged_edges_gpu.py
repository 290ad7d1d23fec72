"""Attention over the paged cache and log probabilities at the ends of their ranges: rows without a place among many rows,
windows without an end, caps far above the scores, logits near the largest value, keys that are no numbers."""
import math

import pytest

torch = pytest.importorskip("torch")

from paged_util import Case, assert_within
from relax_b200 import B200Error, ops

pytestmark = pytest.mark.gpu


def attention(c, **kw):
    out = torch.full((c.tokens, c.heads, c.dim), float("nan"), dtype=c.q.dtype, device="cuda")
    kw = {n: torch.tensor(v, dtype=torch.int32 if n == "prefix" else torch.float32).cuda() if n in ("prefix", "slopes") and v is not None else v
          for n, v in kw.items()}
    ops.paged_attention(c.q, *c.args(), starts=c.starts, max_query=max(c.new), out=out, **kw)
    torch.cuda.synchronize()
    return out


FORMS = [dict(), dict(cap=9.0), dict(slopes=[2.0 ** -(i + 2) for i in range(8)]), dict(cap=9.0, slopes=[2.0 ** -(i + 2) for i in range(8)])]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("new,length,kv", [([300], [200], 2), ([150], [20], 2), ([200, 40, 33], [150, 43, 0], 2), ([70], [66], 8), ([9, 150], [4, 149], 1)])
def test_many_rows_without_a_place_are_zero(cuda_lib, new, length, kv, form):
    """More rows than the sequence has tokens, in the kernel for many rows: those before its beginning see nothing, whatever the mask."""
    c = Case(new, [n - m for n, m in zip(length, new)], 8, kv)
    nowhere = torch.cat([torch.arange(m) < m - n for n, m in zip(length, new)])
    for mask in (dict(), dict(causal=False), dict(prefix=[130] * len(new)), dict(prefix=[1000] * len(new)), dict(window=50, prefix=[129] * len(new))):
        out = attention(c, **form, **mask)
        assert (out[nowhere.cuda()] == 0).all(), (mask, "rows without a place")
        assert_within(out, c.reference(**form, **mask), str(mask))


@pytest.mark.parametrize("new,past", [([1, 1, 1], [300, 0, 40]), ([60, 1, 200], [300, 2, 0]), ([5, 2], [-3, 20]), ([200, 70], [-50, 600])])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 200, 2 ** 33, 2 ** 32 + 5])
def test_a_window_without_an_end(cuda_lib, new, past, window):
    """Windows near the largest whole number, and beyond it, hide nothing: the same bits as without one."""
    c = Case(new, past, 8, 2)
    want = attention(c)
    assert_within(want, c.reference())
    assert torch.equal(attention(c, window=window), want)
    want = attention(c, prefix=[9] * len(new))
    assert torch.equal(attention(c, window=window, prefix=[9] * len(new)), want)


def test_a_window_that_is_no_number_of_tokens(cuda_lib):
    c = Case([1], [30], 4, 2)
    for window in (-1, -2 ** 31, -2 ** 32 + 5):
        with pytest.raises(ValueError, match="window"):
            attention(c, window=window)


def test_what_a_call_that_gave_up_leaves_behind(cuda_lib):
    """Counters of tiles that were cut, left half counted as by a call in which a wait ran out, do not reach the next call."""
    c = Case([140], [6000], 8, 2)
    scratch = ops.paged_attention_scratch("cuda")
    want = attention(c, scratch=scratch)
    assert_within(want, c.reference())
    for left in range(1, 24):                              # (one less than its parts: the first part that arrives would be taken for the last)
        counters = scratch[8192:8192 + 8 * 1016].view(torch.int64)
        assert (counters != 0).any()
        counters.fill_((int(counters.max()) >> 32 << 32) + left)
        scratch[16384:].view(torch.float32).fill_(float("nan"))     # (what a tile that is joined too early reads)
        assert torch.equal(attention(c, scratch=scratch), want), left
    few = Case([1, 1], [3000, 50], 8, 2)                   # the other kernel, in the same memory
    assert_within(attention(few, scratch=scratch), few.reference())
    assert torch.equal(attention(c, scratch=scratch), want)


@pytest.mark.parametrize("cap", [1e3, 1e4, 1e6, 1e9, 1e30])
@pytest.mark.parametrize("new,past,dim,dtype", [([1, 1], [300, 40], 128, "fp16"), ([3], [90], 64, "bf16"), ([60, 5], [300, 0], 128, "fp16"), ([300], [0], 64, "bf16")])
@pytest.mark.parametrize("more", [dict(), dict(window=33, prefix=[2, 2]), dict(slopes=[2.0 ** -(i + 2) for i in range(8)])])
def test_a_cap_far_above_the_scores_changes_little(cuda_lib, cap, new, past, dim, dtype, more):
    """The value is the definition's, with the cap; the bound that of scores without one: tanh of a small number is exact to fp32."""
    c = Case(new, past, 8, 2, dim, 16, dtype)
    c.q.mul_(8.0)
    if "prefix" in more:
        more = {**more, "prefix": more["prefix"][:len(new)]}
    out = attention(c, cap=cap, **more)
    assert_within(out, (c.reference(cap=cap, **more)[0], c.reference(**more)[1]))


@pytest.mark.parametrize("scale", [None, -0.2])
@pytest.mark.parametrize("new,past", [([1, 1, 4], [300, 40, 20]), ([60, 5], [300, 0])])
def test_scores_below_and_above_a_cap(cuda_lib, new, past, scale):
    """Both forms of tanh in one block of keys, and blocks of one of them."""
    c = Case(new, past, 8, 2)
    for factor in (0.5, 4.0, 16.0):
        c.q.mul_(factor)
        for more in (dict(), dict(window=40, prefix=[3] * len(new)), dict(slopes=[2.0 ** -(i + 2) for i in range(8)])):
            assert_within(attention(c, cap=20.0, scale=scale, **more), c.reference(cap=20.0, scale=scale, **more), f"{factor} {more}")


def test_caps_that_are_refused(cuda_lib):
    c = Case([1], [30], 4, 2)
    for cap in (-1.0, float("nan"), float("inf"), 1e31):
        with pytest.raises(B200Error, match="cap"):
            attention(c, cap=cap)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [40, 5000, 70001])
def test_entropy_of_logits_near_the_largest_value(cuda_lib, dtype, V):
    """A distance beyond fp32's range (in the exponent of 2) is a weight of zero, not zero times infinity."""
    big = 3e38
    x = torch.zeros((6, V), dtype=dtype, device="cuda")
    x[0, 7] = big
    x[1, 7], x[1, 9], x[1, 11] = big, -big, float("-inf")
    x[2] = big
    x[3, ::2] = big
    x[4] = -big
    x[4, 5] = big
    x[5] = float(torch.finfo(dtype).min)
    x[5, 5:9] = float(torch.finfo(dtype).max)
    said = ops.token_logprobs(x, torch.full((6,), 7, dtype=torch.int32).cuda(), top=2)
    even = (V + 1) // 2
    want = torch.tensor([0.0, 0.0, math.log(V), math.log(even), 0.0, math.log(4)], dtype=torch.float64)
    assert ((said.entropy.double().cpu() - want).abs() <= 2.0 ** -19 * (1 + want)).all(), said.entropy
    sure = torch.tensor([0.0, 0.0, -math.log(V), 0.0, 0.0, -math.log(4)], dtype=torch.float64)
    for r in (0, 1, 2, 5):
        assert abs(float(said.logprob[r]) - sure[r]) <= 2.0 ** -20 * (1 + abs(sure[r]))
    assert said.top_token[:, 0].tolist() == [7, 7, 0, 0, 5, 5]


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("new,past", [([1, 1], [300, 40]), ([40], [100])])
def test_the_stride_of_a_single_entry_says_nothing(cuda_lib, monkeypatch, native, new, past):
    """One key head, one query head, one page: views whose strides of these dimensions are any numbers."""
    if not native:
        monkeypatch.setattr(ops, "_native", False)
        monkeypatch.setattr(ops, "_torch_call", lambda: False)
    c = Case(new, past, 1, 1)
    want = attention(c)
    c.k, c.v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (c.k, c.v))     # pages by token, then head
    c.q = c.q.as_strided(c.q.shape, (128, 7, 1))
    assert c.k.stride(1) != 16 * 128 and c.q.stride(1) != 128
    assert torch.equal(attention(c), want)
    short = Case([1], [9], 2, 2, ragged=False)
    want = attention(short)
    page = short.table[0, :1].long()
    short.k, short.v = (t[page][0].as_strided((1, 2, 16, 128), (3, 2048, 128, 1)) for t in (short.k, short.v))
    short.table = torch.zeros((1, 1), dtype=torch.int32, device="cuda")
    assert torch.equal(attention(short), want)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("new,past,dim,dtype", [([1, 1], [300, 40], 128, "fp16"), ([3], [90], 64, "bf16"), ([200], [0], 128, "fp16"), ([40], [2000], 64, "bf16"), ([140], [6000], 128, "fp16")])
def test_a_broken_key_is_not_passed_over(cuda_lib, new, past, dim, dtype, bad):
    """Rows that see a key with a NaN or an infinity in it come out as NaN, wherever in a block it lies; rows that do not see it are as they were."""
    c = Case(new, past, 8, 2, dim, 16, dtype)
    position = torch.cat([torch.arange(n, n + m) for n, m in zip(past, new)])
    first = c.starts_list[:-1]
    for at in list(range(min(c.length[0], 34))) + [c.length[0] // 2]:
        where = (int(c.table[0, at // 16]), slice(None), at % 16)
        kept = c.k[where].clone()
        c.k[where] = bad
        for more in (dict(), dict(slopes=[2.0 ** -(i + 2) for i in range(8)]), dict(window=max(new) + 3), dict(cap=20.0)):
            if more.get("cap") and bad == float("inf"):
                continue                                        # (the cap makes it a number)
            sees = position[:new[0]] >= at
            if "window" in more:
                sees &= position[:new[0]] - at < more["window"]
            out = attention(c, **more)[:new[0]].cpu()
            assert torch.isnan(out[sees]).all(), (at, more)
            assert torch.isfinite(out[~sees]).all(), (at, more)
        c.k[where] = kept
