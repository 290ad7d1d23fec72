"""ops.paged_rope_append over pages of 8 bits: what is stored against the 64-bit value, and what earlier tokens become."""
import math

import pytest
import torch

from paged8_util import E4M3, power_for
from paged_util import DTYPES, UNIT
from relax_b200 import ops

pytestmark = pytest.mark.gpu


class Cache:
    def __init__(self, batch, width, kv, dim, page, seed):
        g = torch.Generator().manual_seed(seed)
        self.kv, self.dim, self.page, pool = kv, dim, page, batch * width + 2
        self.table = torch.randperm(pool, generator=g)[: batch * width].view(batch, width).int().cuda()
        self.k, self.v = (torch.full((pool, kv, page, dim), 0x7f, dtype=torch.uint8).cuda().view(E4M3) for _ in "kv")
        self.k_scales, self.v_scales = (torch.full((pool, kv, page // 16), math.nan, dtype=torch.float16).cuda() for _ in "kv")
        self.lengths = [0] * batch

    def state(self):
        return {n: getattr(self, n).cpu().clone() for n in ("k", "v", "k_scales", "v_scales")}


def expected(c, qkv, counts, cos, sin, interleaved, positions=None):
    """(q, k, v) of the rows in 64 bits, and (sequence, position) of each."""
    kv, dim, half = c.kv, c.dim, cos.shape[1]
    x = qkv.double().cpu().view(qkv.shape[0], -1, dim).clone()
    heads = x.shape[1] - 2 * kv
    where = [(b, c.lengths[b] + i) for b, n in enumerate(counts) for i in range(n)]
    for r, (_, t) in enumerate(where):
        at = t if positions is None else positions[r]
        co, si = cos[at].double().cpu(), sin[at].double().cpu()
        part = x[r, : heads + kv]
        a, b = (part[:, 0:2 * half:2], part[:, 1:2 * half:2]) if interleaved else (part[:, :half], part[:, half:2 * half])
        first, second = a * co - b * si, b * co + a * si
        a.copy_(first), b.copy_(second)
    return x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:], where


def call(c, counts, heads, dtype, rotary, interleaved, seed, size=1.0, ragged=True, positions=None):
    g = torch.Generator().manual_seed(seed)
    T = DTYPES[dtype]
    tokens = sum(counts)
    qkv = (torch.randn((tokens, (heads + 2 * c.kv) * c.dim), generator=g) * size).to(T).cuda()
    angle = torch.rand((max(c.lengths) + max(counts) + 9, rotary // 2), generator=g, dtype=torch.float64) * 7
    cos, sin = torch.cos(angle).float().cuda(), torch.sin(angle).float().cuda()
    before = c.state()
    lengths = [a + b for a, b in zip(c.lengths, counts)]
    starts = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32, device="cuda") if ragged else None
    at = None if positions is None else torch.tensor(positions, dtype=torch.int32, device="cuda")
    q = ops.paged_rope_append(qkv, cos, sin, c.k, c.v, c.table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), starts=starts, interleaved=interleaved,
                              positions=at, k_scales=c.k_scales, v_scales=c.v_scales)
    want_q, want_k, want_v, where = expected(c, qkv, counts, cos, sin, interleaved, positions)
    u = UNIT[dtype]
    # q: fp32 products and a sum (3 steps of the larger product), one rounding
    big = qkv.double().cpu().view(tokens, -1, c.dim).abs().amax()
    slack = 2.0 ** -22 * big
    tiny = 2.0 ** -25 if dtype == "fp16" else 0.0
    assert ((q.double().cpu() - want_q).abs() <= u * want_q.abs() + slack + tiny).all()
    after = c.state()
    touched = {"k": torch.zeros(c.k.shape, dtype=torch.bool), "v": torch.zeros(c.k.shape, dtype=torch.bool)}
    blocks = {}
    for r, (b, t) in enumerate(where):
        blocks.setdefault((b, t // 16), []).append((r, t))
    for (b, block), rows in blocks.items():
        page, sub = int(c.table[b, block * 16 // c.page]), block * 16 % c.page // 16
        first = rows[0][1] % 16
        for name, want in (("k", want_k), ("v", want_v)):
            scales, was_scales = after[name + "_scales"], before[name + "_scales"]
            for h in range(c.kv):
                y = want[[r for r, _ in rows], h]
                scale, was = float(scales[page, h, sub]), float(was_scales[page, h, sub])
                most = float(y.abs().max())
                slip = u * most + float(slack) + tiny        # rounded to 16 bits before
                powers = {power_for(max(most - slip, 0)), power_for(most + slip)}
                possible = {2.0 ** p if not first else max(2.0 ** p, was) for p in powers}
                assert scale in possible, (scale, possible, was)
                old = before[name][page, h].double()[sub * 16: sub * 16 + first]
                new = after[name][page, h].double()[sub * 16: sub * 16 + first]
                touched[name][page, h, sub * 16: sub * 16 + first] = True
                if first:
                    moved = old * was                        # exact, but for the smallest steps of the new scale
                    assert ((new * scale - moved).abs() <= torch.where(moved.abs() >= 2.0 ** -6 * scale, 0.0, 2.0 ** -10 * scale)).all()
                for (r, t), value in zip(rows, y):
                    code = after[name][page, h, sub * 16 + t % 16].double()
                    touched[name][page, h, sub * 16 + t % 16] = True
                    held = value.clamp(-448 * scale, 448 * scale)
                    bound = 2.0 ** -4 * value.abs() + 2.0 ** -10 * scale + (u * value.abs() + slack + tiny) * (1 + 2.0 ** -4)
                    assert ((code * scale - held).abs() <= bound).all()
    for name in "kv":                            # everything else is as it was
        assert torch.equal(after[name].view(torch.uint8)[~touched[name]], before[name].view(torch.uint8)[~touched[name]])
    c.lengths = lengths
    return q


@pytest.mark.parametrize("dtype", ("fp16", "bf16"))
@pytest.mark.parametrize("interleaved", (False, True))
@pytest.mark.parametrize("dim,rotary", ((128, 128), (128, 32), (128, 80), (64, 64), (64, 16)))
@pytest.mark.parametrize("page", (16, 64))
def test_prompts_then_tokens(cuda_lib, dim, rotary, interleaved, page, dtype):
    c = Cache(4, 160 // page + 1, 3, dim, page, seed=dim + rotary)
    call(c, [1, 15, 40, 17], 5, dtype, rotary, interleaved, seed=1)
    for i, size in enumerate((1.0, 0.1, 9.0)):   # scales that stay and scales that grow
        call(c, [1, 1, 1, 1], 5, dtype, rotary, interleaved, seed=2 + i, size=size, ragged=i % 2 == 0)
    call(c, [5, 0, 33, 16], 5, dtype, rotary, interleaved, seed=9, size=3.0)


@pytest.mark.parametrize("heads,kv", ((1, 1), (8, 8), (40, 8), (7, 1), (12, 20)))
def test_heads(cuda_lib, heads, kv):
    c = Cache(3, 5, kv, 128, 32, seed=heads)
    call(c, [33, 1, 16], heads, "fp16", 128, False, seed=3)
    call(c, [1, 1, 1], heads, "fp16", 128, False, seed=4, ragged=False)


@pytest.mark.parametrize("dtype,size", (("fp16", 2.0 ** -12), ("fp16", 2000.0), ("fp16", 14000.0), ("bf16", 2.0 ** -40), ("bf16", 2.0 ** 9), ("bf16", 2.0 ** 30)))
def test_very_small_and_very_large_values(cuda_lib, dtype, size):
    c = Cache(2, 3, 2, 64, 16, seed=5)
    call(c, [17, 3], 2, dtype, 64, False, seed=5, size=size)
    call(c, [1, 1], 2, dtype, 64, False, seed=6, size=size)


def test_scales_grow_token_by_token(cuda_lib):
    c = Cache(1, 3, 1, 128, 16, seed=6)
    for i in range(20):
        call(c, [1], 1, "fp16", 128, False, seed=i, size=2.0 ** (i - 12), ragged=False)


def test_positions_of_their_own(cuda_lib):
    c = Cache(2, 4, 2, 64, 16, seed=7)
    call(c, [6, 9], 3, "fp16", 64, False, seed=7, positions=[2, 2, 0, 5, 1, 3, 8, 7, 6, 5, 4, 3, 2, 1, 0])


def test_what_is_not_finite(cuda_lib):
    c = Cache(1, 2, 1, 64, 16, seed=8)
    qkv = torch.ones((3, 3 * 64), dtype=torch.float16, device="cuda")
    qkv[0, 64], qkv[1, 130], qkv[2, 131] = math.inf, math.nan, -math.inf
    cos, sin = torch.ones((4, 8), device="cuda"), torch.zeros((4, 8), device="cuda")
    ops.paged_rope_append(qkv, cos, sin, c.k, c.v, c.table, torch.tensor([3], dtype=torch.int32, device="cuda"),
                          starts=torch.tensor([0, 3], dtype=torch.int32, device="cuda"), k_scales=c.k_scales, v_scales=c.v_scales)
    page = c.table[0, 0].long()
    k, v = c.k[page, 0, :3].float().cpu(), c.v[page, 0, :3].float().cpu()
    assert float(c.k_scales[page, 0, 0]) == float(c.v_scales[page, 0, 0]) == 2.0 ** -8      # of ones
    assert torch.isnan(k[0, 0]) and torch.isnan(v[1, 2]) and torch.isnan(v[2, 3])
    assert (k[1:] == 256).all() and int(torch.isnan(v).sum()) == 2
    zero = torch.zeros((1, 3 * 64), dtype=torch.float16, device="cuda")
    ops.paged_rope_append(zero, cos, sin, c.k, c.v, c.table, torch.tensor([17], dtype=torch.int32, device="cuda"), k_scales=c.k_scales, v_scales=c.v_scales)
    page = c.table[0, 1].long()
    assert float(c.k_scales[page, 0, 0]) == 2.0 ** -24 and (c.k[page, 0, 0].float() == 0).all()


def test_rows_without_a_place(cuda_lib):
    c = Cache(2, 2, 1, 64, 16, seed=9)
    before = c.state()
    qkv = torch.ones((4, 3 * 64), dtype=torch.float16, device="cuda")
    cos, sin = torch.ones((9, 32), device="cuda"), torch.zeros((9, 32), device="cuda")
    q = ops.paged_rope_append(qkv, cos, sin, c.k, c.v, c.table, torch.tensor([1, 0], dtype=torch.int32, device="cuda"),
                              starts=torch.tensor([0, 3, 4], dtype=torch.int32, device="cuda"), k_scales=c.k_scales, v_scales=c.v_scales)
    assert (q[:2] == 0).all() and (q[2] == 1).all() and (q[3] == 0).all()
    after = c.state()
    changed = (after["k"].view(torch.uint8) != before["k"].view(torch.uint8)).flatten(1).any(dim=1).nonzero().flatten().tolist()
    assert changed == [int(c.table[0, 0])]


def test_streams_graphs_and_strides(cuda_lib):
    got = []
    for way in range(3):
        c = Cache(3, 4, 2, 128, 16, seed=10)
        g = torch.Generator(device="cuda").manual_seed(11)
        wide = torch.randn((30, 6 * 128 + 8), device="cuda", generator=g).half()
        qkv = wide[:, : 6 * 128]
        angle = torch.rand((40, 64), device="cuda", generator=g)
        args = (angle.cos().contiguous(), angle.sin().contiguous(), c.k, c.v, c.table, torch.tensor([20, 7, 3], dtype=torch.int32, device="cuda"))
        kw = dict(starts=torch.tensor([0, 20, 27, 30], dtype=torch.int32, device="cuda"), k_scales=c.k_scales, v_scales=c.v_scales)
        if way == 0:
            q = ops.paged_rope_append(qkv.contiguous(), *args, **kw)
        elif way == 1:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                q = ops.paged_rope_append(qkv, *args, **kw)
            side.synchronize()
        else:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                q = ops.paged_rope_append(qkv, *args, **kw)
            graph.replay()
            graph.replay()                       # the same call again changes nothing
        got.append({**c.state(), "q": q.cpu()})
    for other in got[1:]:
        for n in got[0]:
            a, b = (t.view(torch.uint8) if t.dtype is E4M3 else t.view(torch.int16) for t in (got[0][n], other[n]))
            assert torch.equal(a, b), n


def test_refusals(cuda_lib):
    c = Cache(2, 2, 2, 64, 16, seed=12)
    qkv = torch.zeros((2, 6 * 64), dtype=torch.float16, device="cuda")
    table = torch.zeros((9, 32), device="cuda")
    good = dict(qkv=qkv, cos=table, sin=table, k_pages=c.k, v_pages=c.v, page_table=c.table, lengths=torch.ones(2, dtype=torch.int32, device="cuda"),
                k_scales=c.k_scales, v_scales=c.v_scales)
    ops.paged_rope_append(**good)
    for bad in (dict(k_scales=None), dict(k_scales=None, v_scales=None), dict(v_scales=c.v_scales.float()), dict(k_scales=c.k_scales[1:]), dict(qkv=qkv.float()),
                dict(k_pages=c.k.view(torch.uint8).to(torch.float16), v_pages=c.v.view(torch.uint8).to(torch.float16)), dict(v_scales=c.v_scales.cpu()),
                dict(sin=table[:, :16])):
        with pytest.raises(ValueError):
            ops.paged_rope_append(**{**good, **bad})
    with pytest.raises(ops.B200Error):
        ops.paged_rope_append(**{**good, "cos": table[:, :4].contiguous(), "sin": table[:, :4].contiguous()})
