"""ops.sample_tokens against its definition in 64 bits.  The token has to be the same: both sides compare sums of weights of fp64, whose
difference (2^-37 of a weight) would have to reach from a random number to the next border."""
import math

import numpy as np
import pytest
import torch

from sample_util import allowed, sample
from relax_b200 import ops

pytestmark = pytest.mark.gpu
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def check(logits, uniform, **how):
    """`how`: numbers, or lists of one for each row."""
    rows = logits.shape[0]
    args = {n: v if not isinstance(v, list) else torch.tensor(v, dtype=torch.int32 if n == "top_k" else torch.float32, device="cuda") for n, v in how.items()}
    got = ops.sample_tokens(logits, uniform, **args)
    x, u = logits.double().cpu().numpy(), uniform.cpu().numpy()
    for i in range(rows):
        token, logprob = sample(x[i], u[i], **{n: v[i] if isinstance(v, list) else v for n, v in how.items()})
        assert int(got.token[i]) == token, f"row {i}: {int(got.token[i])} instead of {token}, u = {u[i]}, {how}"
        value = float(got.logprob[i])
        if math.isfinite(logprob):                # one rounding to fp32; the weight and the sum are 2^-37 exact each
            assert abs(value - logprob) <= 2.0 ** -24 * abs(logprob) + 2.0 ** -36, f"row {i}"
        else:
            assert math.isnan(value) == math.isnan(logprob) and (math.isnan(value) or value == logprob)
    return got


def logits_of(rows, V, dtype, seed, size=2.5, stride=0, offset=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    flat = torch.full((rows * (V + stride) + offset,), float("nan"), dtype=DTYPES[dtype], device="cuda")
    x = flat[offset:].view(rows, V + stride)[:, :V]
    x.copy_(torch.randn((rows, V), device="cuda", generator=g) * size)
    return x, torch.rand(rows, device="cuda", generator=g)


SETTINGS = (dict(), dict(temperature=0.7), dict(top_k=50), dict(top_k=1), dict(top_p=0.9), dict(min_p=0.05), dict(temperature=1.3, top_k=400, top_p=0.8, min_p=0.01),
            dict(temperature=0.0), dict(top_p=0.0), dict(top_p=0.999), dict(top_k=10 ** 6), dict(min_p=1.0), dict(min_p=7.0), dict(top_k=3, top_p=0.5))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("how", SETTINGS, ids=lambda h: "-".join(f"{n}{v}" for n, v in h.items()) or "plain")
@pytest.mark.parametrize("rows,V", ((1, 1), (3, 2), (5, 7), (4, 1000), (2, 4097), (1, 32000), (37, 2049)))
def test_settings(cuda_lib, rows, V, how, dtype):
    check(*logits_of(rows, V, dtype, seed=rows * 7 + V), **how)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V", ((1, 151999), (9, 152000), (300, 5003)))
def test_rows_of_their_own_settings(cuda_lib, rows, V, dtype):
    pick = np.random.default_rng(rows)
    check(*logits_of(rows, V, dtype, seed=V), temperature=pick.choice([0.0, 0.5, 1.0, 1.4], rows).tolist(), top_k=pick.choice([0, 1, 7, 300, 5000], rows).tolist(),
          top_p=pick.choice([1.0, 0.3, 0.95, 0.9999], rows).tolist(), min_p=pick.choice([0.0, 0.02, 0.5], rows).tolist())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset,stride", ((0, 0), (1, 3), (5, 0), (3, 13)))
def test_rows_that_begin_anywhere(cuda_lib, dtype, offset, stride):
    check(*logits_of(6, 1003, dtype, seed=offset, offset=offset, stride=stride), top_k=100, top_p=0.9)
    check(*logits_of(6, 9001, dtype, seed=offset, offset=offset, stride=stride))


@pytest.mark.parametrize("how", (dict(), dict(top_k=1000), dict(top_p=0.5), dict(top_k=2500, top_p=0.25), dict(min_p=0.5), dict(top_p=0.5, min_p=1.0)))
@pytest.mark.parametrize("V", (64, 5000, 40000))
def test_equal_logits(cuda_lib, V, how):
    """Whole numbers of equal weights: the lowest indices stay."""
    _, u = logits_of(5, 8, "fp32", seed=1)
    check(torch.full((5, V), 3.25, device="cuda"), u, **how)
    two = torch.full((5, V), -1.0, device="cuda", dtype=torch.bfloat16)
    two[:, ::3] = -0.5
    check(two, u, **how)
    zeros = torch.zeros((5, V), device="cuda")
    zeros[:, 1::2] = -0.0                        # one value
    check(zeros, u, **how)


@pytest.mark.parametrize("temperature", (1e-6, 1e-38, 0.01, 100.0, 1e30, math.inf))
@pytest.mark.parametrize("how", (dict(), dict(top_k=20), dict(top_p=0.7), dict(min_p=0.3)))
def test_far_temperatures(cuda_lib, temperature, how):
    check(*logits_of(4, 6001, "fp32", seed=3), temperature=temperature, **how)


@pytest.mark.parametrize("how", (dict(), dict(top_k=20), dict(top_p=0.7), dict(temperature=0.0), dict(min_p=0.3)))
@pytest.mark.parametrize("V", (5, 33000))
def test_excluded_entries(cuda_lib, V, how):
    x, u = logits_of(7, V, "fp16", seed=5)
    x[0, : V // 2] = -math.inf
    x[1] = -math.inf
    x[1, V - 1] = -60000.0
    x[2] = -math.inf
    x[3, 1] = math.nan
    x[4, V - 2] = math.inf
    x[5] = -math.inf
    x[5, 2:4] = 1.0
    x[6, 1] = 65504.0
    check(x, u, **how)


def test_the_ends_of_the_random_numbers(cuda_lib):
    x, _ = logits_of(8, 3001, "fp32", seed=6)
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, 1.5, -0.5, 1e-30, math.nan, 0.5], device="cuda")
    got = check(x[:6], u[:6].contiguous())
    assert int(got.token[0]) == 0 and int(got.token[2]) == 3000
    check(x, torch.where(u.isnan(), -1.0, u), top_k=10)
    assert int(ops.sample_tokens(x, u, top_k=10).token[6]) == int(allowed(x[6].double().cpu().numpy(), top_k=10)[0][0])


def test_far_apart_values(cuda_lib):
    x = torch.tensor([[3e38, -3e38, 3e38, 0.0, -math.inf], [1.0, 1.0 + 2.0 ** -23, 1.0, 1.0, 1.0]], device="cuda")
    u = torch.tensor([0.7, 0.3], device="cuda")
    for how in (dict(), dict(top_k=1), dict(top_k=2), dict(top_p=0.5), dict(min_p=0.5)):
        check(x, u, **how)


def test_many_draws_follow_the_distribution(cuda_lib):
    """20000 draws of one row: counts within five standard deviations of the probabilities."""
    x, _ = logits_of(1, 50, "fp32", seed=8)
    n = 20000
    u = torch.rand(n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(9))
    got = ops.sample_tokens(x.expand(n, 50).contiguous(), u, temperature=0.9, top_p=0.9)
    keep, w = allowed(x[0].double().cpu().numpy(), temperature=0.9, top_p=0.9)
    counts = np.bincount(got.token.cpu().numpy(), minlength=50)
    assert counts.sum() == counts[keep].sum() == n
    p = w / w.sum()
    assert (np.abs(counts[keep] - n * p) <= 5 * np.sqrt(n * p * (1 - p)) + 1).all()


def test_streams_graphs_and_repetition(cuda_lib):
    x, u = logits_of(33, 32000, "fp16", seed=10)
    want = ops.sample_tokens(x, u, top_k=40, top_p=0.95, temperature=0.8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.sample_tokens(x, u, top_k=40, top_p=0.95, temperature=0.8)
    side.synchronize()
    assert torch.equal(other.token, want.token) and torch.equal(other.logprob, want.logprob)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ops.sample_tokens(x, u, top_k=40, top_p=0.95, temperature=0.8)
    x.copy_(x.flip(0).clone())
    u.copy_(u.flip(0).clone())
    graph.replay()
    assert torch.equal(held.token, want.token.flip(0)) and torch.equal(held.logprob, want.logprob.flip(0))


def test_refusals(cuda_lib):
    x, u = logits_of(3, 100, "fp16", seed=11)
    for bad in (dict(uniform=u[:2]), dict(uniform=u.double()), dict(temperature=torch.ones(2, device="cuda")), dict(top_k=torch.ones(3, device="cuda")),
                dict(top_p=torch.ones(3, dtype=torch.float64, device="cuda")), dict(min_p=torch.ones(3)), dict(logits=x.t()), dict(logits=x.int()),
                dict(logits=x[0])):
        with pytest.raises(ValueError):
            ops.sample_tokens(**{**dict(logits=x, uniform=u), **bad})
    with pytest.raises(ops.B200Error):
        ops.sample_tokens(x.expand(3, 100).as_strided((3, 100), (50, 1)), u)
    empty = ops.sample_tokens(x[:0], u[:0])
    assert empty.token.shape == empty.logprob.shape == (0,)


@pytest.mark.parametrize("V", (3000, 40000, 152000))
@pytest.mark.parametrize("top_p,min_p", ((0.95, 0.001), (0.95, 0.02), (0.5, 0.0005), (0.9, 0.15), (0.999, 1e-6), (0.3, 1.0)))
@pytest.mark.parametrize("top_k", (0, 700, 2500))
def test_whichever_border_is_the_higher_one(cuda_lib, V, top_p, min_p, top_k):
    """top_p's and min_p's borders on either side of each other, and near each other, with all of top_k's ways."""
    check(*logits_of(5, V, "fp32", seed=V + top_k), top_p=top_p, min_p=min_p, top_k=top_k)
    check(*logits_of(3, V, "bf16", seed=V + top_k), top_p=top_p, min_p=min_p, top_k=top_k, temperature=0.4)
