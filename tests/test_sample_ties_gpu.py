"""ops.sample_tokens where many logits are the same: weights are equal to the bit, so that borders among ties lie where whole numbers say."""
import math

import numpy as np
import pytest
import torch

from relax_b200 import ops
from test_sample_gpu import check, logits_of

pytestmark = pytest.mark.gpu


def ties(rows, V, n, value, seed):
    """n entries of each row are `value`; the others count as excluded (2000 below it, more than 690 temperatures) or are.  (Weights of 10^-17 would be an
    ill-posed question: in 64 bits their sum beside that of the ties hangs on its order.)"""
    pick = np.random.default_rng(seed)
    x = torch.full((rows, V), value - 2000.0)
    for r in range(rows):
        x[r, pick.choice(V, n, replace=False)] = value
        x[r, pick.choice(V, V // 9, replace=False)].clamp_(max=-math.inf if r % 2 else value - 2000.0)
    return x.cuda(), torch.from_numpy(pick.random(rows, dtype=np.float32)).cuda()


@pytest.mark.parametrize("temperature", (1.0, 0.7, 0.8, 0.1, 2.5))
@pytest.mark.parametrize("value", (3.25, 7.75, 27.25, -11.3))
@pytest.mark.parametrize("n,V", ((100, 130), (400, 1000), (600, 33000)))
def test_top_p_among_ties(cuda_lib, n, V, value, temperature):
    """top_p n is a whole number, or the half of one: so many of n equal entries stay, with top_k's list and without."""
    x, u = ties(4, V, n, value, seed=n)
    for top_p in (0.75, 0.5, 0.25, 0.125):
        check(x, u, temperature=temperature, top_p=top_p, top_k=n)
        check(x, u, temperature=temperature, top_p=top_p)


@pytest.mark.parametrize("temperature", (0.7, 0.1))
@pytest.mark.parametrize("V", (100, 640))
def test_a_draw_among_ties(cuda_lib, V, temperature):
    """Where u V is a whole number, the weights up to the entry before are u times all, which is not more."""
    x = torch.full((V, V), 7.75, device="cuda")
    u = torch.arange(V, device="cuda").float() / V
    for how in (dict(), dict(top_k=V - 1)):
        kept = V if not how else V - 1
        got = ops.sample_tokens(x, u, temperature=temperature, **how).token.cpu()
        want = torch.tensor([math.floor(float(v) * kept) for v in u.tolist()])
        assert torch.equal(got.long(), want)


@pytest.mark.parametrize("min_p", (0.3, 1.0, 7.0))
@pytest.mark.parametrize("V", (50, 6001))
def test_an_infinite_temperature_makes_all_weights_the_largest(cuda_lib, V, min_p):
    x, u = logits_of(3, V, "fp32", seed=V)
    for how in (dict(), dict(top_k=20), dict(top_p=0.5)):
        check(x, u, temperature=math.inf, min_p=min_p, **how)
