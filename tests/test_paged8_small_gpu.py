"""ops.paged_attention over 8-bit pages whose scales are so small that code times scale is no number of fp16: calls of many rows and of few give the definition."""
import pytest
import torch

import paged_util
from paged8_util import E4M3, Case8, to_e4m3
from relax_b200 import ops

pytestmark = pytest.mark.gpu


def refill(case, name, powers, size, seed):
    """Codes of normal numbers times `size`, every block's scale one of 2^powers."""
    g = torch.Generator().manual_seed(seed)
    codes, scales, table = getattr(case, name + "8").cpu().view(torch.uint8), getattr(case, name + "_scales").cpu(), case.table.cpu()
    held = case.keys if name == "k" else case.values
    for b, n in enumerate(case.length):
        for i in range(0, n, 16):
            at, rows = int(table[b, i // case.page]), min(16, n - i)
            code = to_e4m3(torch.randn((case.kv, rows, case.dim), generator=g, dtype=torch.float64) * size)
            power = torch.tensor(powers)[torch.randint(len(powers), (case.kv,), generator=g)]
            codes[at, :, i % case.page:i % case.page + rows] = code.to(E4M3).view(torch.uint8)
            scales[at, :, i % case.page // 16] = torch.exp2(power.double()).half()
            held[b][:, i:i + rows] = code * torch.exp2(power.double())[:, None, None]
    setattr(case, name + "8", codes.view(E4M3).cuda())
    setattr(case, name + "_scales", scales.cuda())


def check(case, **kw):
    """Within the bound of 16 bits without its room for numbers below fp16's: of a result one rounding in bf16 (in fp16 at least half its smallest
    step), of a weight two by fp16, the second by up to 2^-9 smaller (2^-25 / 2^-9 of the largest weight each at most)."""
    got = ops.paged_attention(case.q, *case.args(), starts=case.starts, max_query=max(case.new + [1]), **case.scales(), **kw)
    torch.cuda.synchronize()
    assert ops._lib.lib().b200_device_error_flags() == 0
    out, bound = paged_util.Case.reference(case, **kw)
    if case.dtype == "bf16":
        bound = bound - 2.0 ** -24
    q = case.q.double().cpu()
    for b, n in enumerate(case.length):
        rows = slice(case.starts_list[b], case.starts_list[b + 1])
        see, _ = case.visible(b, window=kw.get("window", 0))
        for h in range(case.heads):
            k, v = (t[b][h // (case.heads // case.kv)] for t in (case.keys, case.values))
            x = q[rows, h] @ k.T * kw.get("scale", case.dim ** -0.5)
            if kw.get("cap"):
                x = kw["cap"] * torch.tanh(x / kw["cap"])
            total = torch.exp(x - x.masked_fill(~see, -1e300).amax(dim=1, keepdim=True)).masked_fill(~see, 0.0).sum(dim=1, keepdim=True)
            bound[rows, h] += 2 * 2.0 ** -16 / total * (see.double() @ v.abs())
    off = (got.double().cpu() - out).abs()
    assert (off <= bound).all(), f"{float(off.max())} of {float(out.abs().max())}, {int((off > bound).sum())} of {off.numel()}"


MIXED = (-24, -23, -20, -16, -15, -14, -9)


@pytest.mark.parametrize("new", (1, 60, 200))
@pytest.mark.parametrize("dim,page", ((128, 16), (128, 64), (64, 32)))
@pytest.mark.parametrize("powers", ((-24,), (-22, -24), MIXED))
def test_small_values(cuda_lib, powers, dim, page, new):
    """bf16 rows hold them.  (With scales of very different sizes a value of the small ones is lost beside the largest, and so it is in the bound.)"""
    case = Case8([new, 3], [300, 77], 4, 2, dim, page, "bf16", seed=new)
    refill(case, "v", powers, 2.0, seed=1)
    check(case)
    check(case, window=33)


@pytest.mark.parametrize("dtype", ("fp16", "bf16"))
@pytest.mark.parametrize("new", (1, 60, 200))
@pytest.mark.parametrize("dim,page", ((128, 16), (64, 128)))
@pytest.mark.parametrize("powers", ((-24,), MIXED[:4]))
@pytest.mark.parametrize("kw", (dict(), dict(window=50), dict(cap=4.0)))
def test_small_keys(cuda_lib, kw, powers, dim, page, new, dtype):
    """Large queries see them: scores of a few units."""
    case = Case8([new, 3], [300, 77], 4, 2, dim, page, dtype, seed=new)
    refill(case, "k", powers, 2.0, seed=2)
    case.q *= 2.0 ** 12
    check(case, scale=2.0 ** -12 * 2.0 ** (-max(powers)) / 4 * dim ** -0.5, **kw)


@pytest.mark.parametrize("new", (60, 300))
@pytest.mark.parametrize("kw", (dict(slopes=[0.02, 0.01, 0.05, 0.0]), dict(slopes=[0.01] * 4, cap=8.0)))
def test_small_keys_and_values_with_a_bias(cuda_lib, kw, new):
    """All of it at once: calls of many rows against the rows one by one, which take codes as they are."""
    case = Case8([new], [150], 4, 2, 128, 16, "bf16", seed=3)
    for name in "kv":
        refill(case, name, (-24, -19), 2.0, seed=4)
    case.q *= 2.0 ** 12
    args = dict(scale=2.0 ** 5 * 128 ** -0.5, **{**kw, "slopes": torch.tensor(kw["slopes"], device="cuda")})
    many = ops.paged_attention(case.q, *case.args(), starts=case.starts, max_query=new, **case.scales(), **args).double()
    for i in (0, 1, new // 2, new - 1):
        few = ops.paged_attention(case.q[i:i + 1], *case.args()[:3], torch.tensor([150 + i + 1], dtype=torch.int32, device="cuda"), **case.scales(), **args).double()
        assert ((many[i] - few[0]).abs() <= 2 * 2.0 ** -8 * few[0].abs() + 2.0 ** -9 * few[0].abs().amax(dim=-1, keepdim=True)).all()


def test_blocks_of_small_scales_among_many_items(cuda_lib):
    """More sequences than CTAs, some short and some long, tiny blocks here and there: every block's rows read its own."""
    past = [(53 * i) % 700 for i in range(180)]
    case = Case8([17 + i % 5 for i in range(180)], past, 2, 1, 64, 16, "bf16", seed=5)
    refill(case, "v", (-24,), 2.0, seed=6)
    refill(case, "k", (-24, -15, -13), 0.25, seed=7)
    case.q *= 2.0 ** 12
    check(case, scale=2.0 ** 3 * 64 ** -0.5)
