"""ops.sample_tokens on long rows whose border lies among more entries than a list holds, on as many CTAs as a row gets, and on few."""
import pytest
import torch

from test_sample_gpu import check, logits_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ("fp32", "bf16"))
@pytest.mark.parametrize("rows", (2, 40))
@pytest.mark.parametrize("size,temperature", ((2.5, 2.5), (2.5, 4.0), (1.0, 1.0), (0.01, 1.0)))
@pytest.mark.parametrize("how", (dict(top_p=0.9), dict(top_p=0.5, min_p=0.2), dict(top_p=0.8, top_k=60000)))
def test_long_flat_rows(cuda_lib, how, size, temperature, rows, dtype):
    check(*logits_of(rows, 152000, dtype, seed=rows, size=size), temperature=temperature, **how)


@pytest.mark.parametrize("V", (131072, 152001))
@pytest.mark.parametrize("how", (dict(top_p=0.5), dict(top_k=1000), dict(top_k=70000, top_p=0.25), dict(min_p=1.0)))
def test_long_equal_rows(cuda_lib, V, how):
    _, u = logits_of(3, 8, "fp32", seed=2)
    x = torch.full((3, V), 7.75, device="cuda")
    x[1, ::2] = 7.5
    x[2, : V // 2] = float("-inf")
    check(x, u, temperature=0.7, **how)


def test_one_row_of_many_is_flat(cuda_lib):
    """64 rows at once, as a served batch has them: the flat one among the others."""
    x, u = logits_of(64, 152000, "fp16", seed=3)
    x[17] *= 0.25
    check(x, u, top_p=0.9, top_k=[0] * 63 + [40])
