"""The new operators through the Python checks (no extension): the same results."""
import pytest
import torch

from paged8_util import Case8
from relax_b200 import ops

pytestmark = pytest.mark.gpu


def test_without_the_extension(cuda_lib, monkeypatch):
    case = Case8([1, 3], [40, 17], 4, 2, seed=1)
    g = torch.Generator(device="cuda").manual_seed(2)
    logits, u = torch.randn((5, 777), device="cuda", generator=g), torch.rand(5, device="cuda", generator=g)
    qkv = torch.randn((4, 8 * 128), device="cuda", generator=g).half()
    angle = torch.rand((64, 64), device="cuda", generator=g)
    i32 = dict(dtype=torch.int32, device="cuda")

    def all_of_them():
        k, v, ks, vs = (t.clone() for t in (case.k8, case.v8, case.k_scales, case.v_scales))
        q = ops.paged_rope_append(qkv, angle.cos(), angle.sin(), k, v, case.table, case.lengths, starts=case.starts, k_scales=ks, v_scales=vs)
        a = ops.paged_attention(q, k, v, case.table, case.lengths, starts=case.starts, max_query=3, k_scales=ks, v_scales=vs)
        plan = ops.paged_plan(torch.full((2, 3), -1, **i32), torch.zeros(2, **i32), torch.tensor([17, 3], **i32), torch.arange(9, **i32),
                              torch.tensor([9], **i32), 16, 24)
        drawn = ops.sample_tokens(logits, u, temperature=torch.full((5,), 0.9, device="cuda"), top_k=50, top_p=0.95, min_p=0.01)
        return [q, a, *plan, *drawn, k.view(torch.uint8), v.view(torch.uint8), ks.view(torch.int16), vs.view(torch.int16)]

    want = all_of_them()
    monkeypatch.setattr(ops, "_native", False)
    monkeypatch.setattr(ops, "_torch_call", lambda: False)
    for a, b in zip(want, all_of_them()):
        assert torch.equal(a, b)
