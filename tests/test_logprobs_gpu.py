"""Log probabilities, entropy and likeliest entries against 64 bits: ties, excluded entries, odd widths and alignments, degenerate rows."""
import math

import pytest

torch = pytest.importorskip("torch")

from relax_b200 import B200Error, _lib, ops

pytestmark = pytest.mark.gpu
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def check(x, tokens, top):
    got = ops.token_logprobs(x, tokens, top=top)
    torch.cuda.synchronize()
    d = x.double().cpu()
    total = torch.logsumexp(d, dim=1)
    rows = torch.arange(x.shape[0])
    p = torch.exp(d - total[:, None])
    want = d[rows, tokens.cpu().long()] - total
    # fp32: the difference to the maximum, a sum of V weights each 2^-22 off in the mean, a logarithm
    slack = 2.0 ** -22 * (1 + want.abs().clamp(max=1e30)) + 2.0 ** -21
    near = (got.logprob.double().cpu() - want).abs() <= slack
    assert (near | (want == got.logprob.double().cpu())).all()
    entropy = total - torch.where(p > 0, p * d, 0.0).sum(dim=1)
    assert ((got.entropy.double().cpu() - entropy).abs() <= 2.0 ** -19 * (1 + entropy.abs())).all()
    if top:
        order = torch.sort(x.float() + 0.0, dim=1, descending=True, stable=True).indices[:, :top].cpu()
        assert torch.equal(got.top_token.cpu().long(), order)
        want = d.gather(1, order) - total[:, None]
        off = (got.top_logprob.double().cpu() - want).abs()
        assert ((off <= 2.0 ** -22 * (1 + want.abs().clamp(max=1e30)) + 2.0 ** -21) | (want == got.top_logprob.double().cpu())).all()
    return got


@pytest.mark.parametrize("rows,V", [(1, 1), (1, 7), (3, 33), (2, 1000), (1, 32000), (5, 32001), (40, 5003), (300, 2049), (1, 151937), (3, 4099)])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_rows(cuda_lib, rows, V, dtype):
    g = torch.Generator().manual_seed(V)
    x = (torch.randn((rows, V), generator=g) * 3).to(DTYPES[dtype]).cuda()
    tokens = torch.randint(0, V, (rows,), generator=g, dtype=torch.int32).cuda()
    for top in sorted({0, 1, min(5, V), min(32, V)}):
        check(x, tokens, top)
    flat = torch.empty(rows * (V + 3) + 1, dtype=x.dtype, device="cuda")
    view = flat[1:].view(rows, V + 3)[:, :V]                    # another alignment in every row
    view.copy_(x)
    check(view, tokens, min(20, V))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("V", [40, 3000, 40000])
def test_ties(cuda_lib, dtype, V):
    """Equal values go by index: few values, one value, more equal ones than the list of candidates holds; both zeros are equal."""
    g = torch.Generator().manual_seed(1)
    tokens = torch.full((4,), V - 1, dtype=torch.int32).cuda()
    for top in (1, 5, 32):
        check(torch.randint(0, 3, (4, V), generator=g).to(DTYPES[dtype]).cuda(), tokens, top)
        check(torch.full((4, V), 1.5, dtype=DTYPES[dtype], device="cuda"), tokens, top)
        x = torch.zeros((4, V), dtype=DTYPES[dtype], device="cuda")
        x[:, ::2] = -0.0
        x[:, V // 2] = 1.0
        check(x, tokens, top)
        x = torch.full((4, V), float(torch.finfo(DTYPES[dtype]).min), dtype=DTYPES[dtype], device="cuda")      # masked by the lowest value
        x[:, V - 3:] = 2.0
        check(x, tokens, top)


def test_large_values_where_one_group_of_threads_looks(cuda_lib):
    """The large values lie 2048 apart, as one group of threads sees them: more than the list of candidates holds."""
    V = 2048 * 700
    x = torch.randn((2, V), generator=torch.Generator().manual_seed(2)).cuda()
    for i in range(8):
        x[:, i::2048] += 50
    check(x, torch.zeros(2, dtype=torch.int32).cuda(), 32)
    check(x[:1], torch.zeros(1, dtype=torch.int32).cuda(), 5)
    many = x[:1].expand(160, V)[:, : 2048 * 600].half()          # one CTA a row
    check(many, torch.zeros(160, dtype=torch.int32).cuda(), 7)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_excluded_entries(cuda_lib, dtype):
    g = torch.Generator().manual_seed(3)
    for V in (50, 5000, 40000):
        for keep in (1, 3, 40):
            x = torch.full((3, V), -math.inf, dtype=DTYPES[dtype])
            at = torch.randperm(V, generator=g)[:keep]
            x[:, at] = torch.randn((3, keep), generator=g).to(x.dtype)
            got = check(x.cuda(), at[:1].int().expand(3).contiguous().cuda(), 20)
            assert torch.isfinite(got.logprob).all()
            other = torch.full((3,), int(next(i for i in range(V) if i not in set(at.tolist()))), dtype=torch.int32).cuda()
            assert (check(x.cuda(), other, 0).logprob == -math.inf).all()


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("V", [40, 20000])
def test_degenerate_rows(cuda_lib, dtype, V):
    x = torch.zeros((5, V), dtype=DTYPES[dtype], device="cuda")
    x[0] = -math.inf
    x[1, 30] = math.nan
    x[2, 7] = math.inf
    x[3, 9] = -math.inf
    x[4, :8] = -math.inf
    x[4, 20] = math.nan
    got = ops.token_logprobs(x, torch.tensor([0, 3, 7, 9, 2], dtype=torch.int32).cuda(), top=4)
    torch.cuda.synchronize()
    assert got.logprob[0] == -math.inf and got.entropy[0] == 0 and (got.top_logprob[0] == -math.inf).all() and got.top_token[0].tolist() == [0, 1, 2, 3]
    for r in (1, 2, 4):
        assert torch.isnan(got.logprob[r]) and torch.isnan(got.entropy[r]) and torch.isnan(got.top_logprob[r]).all()
        assert got.top_token[r].tolist() == [0, 1, 2, 3]
    assert got.logprob[3] == -math.inf and abs(float(got.entropy[3]) - math.log(V - 1)) < 1e-5
    far = ops.token_logprobs(x[3:4], torch.tensor([V], dtype=torch.int32).cuda())
    assert far.logprob[0] == -math.inf and far.top_token is None
    assert ops.token_logprobs(x[3:4], torch.tensor([-1], dtype=torch.int32).cuda()).logprob[0] == -math.inf


def test_a_common_offset_costs_nothing(cuda_lib):
    x = torch.randn((4, 3000), generator=torch.Generator().manual_seed(4)).mul(8).round().div(8).cuda()
    t = torch.arange(4, dtype=torch.int32).cuda()
    a, b = check(x, t, 3), check(x + 4096.0, t, 3)
    assert torch.equal(a.logprob, b.logprob) and torch.equal(a.entropy, b.entropy)


def test_refusals(cuda_lib):
    x = torch.zeros((2, 100), dtype=torch.float16, device="cuda")
    t = torch.zeros(2, dtype=torch.int32, device="cuda")
    for a, b, kw in ((x.double(), t, {}), (x[0], t, {}), (x.t(), t, {}), (x, t.long(), {}), (x, t[:1], {}), (x, t.cpu(), {}), (x, t, dict(top=33)),
                     (x[:, :3], t, dict(top=4)), (x, t, dict(top=-1)), (x[:, :0], t, {}), (x.cpu(), t.cpu(), {})):
        with pytest.raises((ValueError, B200Error, RuntimeError)):
            ops.token_logprobs(a, b, **kw)
    assert ops.token_logprobs(x[:0], t[:0], top=3).top_token.shape == (0, 3)
    p = x.data_ptr()
    call = cuda_lib.b200_token_logprobs
    assert call(p, 3, 100, p, p, p, None, None, 2, 100, 0, 0) == _lib.EINVAL
    assert call(p + 1, 0, 100, p, p, p, None, None, 2, 100, 0, 0) == _lib.EINVAL
    assert call(p, 0, 50, p, p, p, None, None, 2, 100, 0, 0) == _lib.EINVAL
    assert call(p, 0, 100, None, p, p, None, None, 2, 100, 0, 0) == _lib.EINVAL
    assert call(p, 0, 100, p, p, p, None, p, 2, 100, 3, 0) == _lib.EINVAL
    assert call(None, 0, 100, p, p, p, None, None, 2, 100, 0, 0) == _lib.EINVAL
