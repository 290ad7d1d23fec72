"""The decoder's cache and logits when a text comes at once and when it comes in parts: 16 bits within the matmuls' rounding, 8 bits block by block."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_paged_decoder_gpu import model
from test_paged8_forget_gpu import held

pytestmark = pytest.mark.gpu
PARTS = ((0, 1), (1, 7), (7, 8), (8, 40), (40, 50))


def both(bits, **kw):
    """(whole, parts): the logits of every token, places 0 and 1 of the decoder, which comes third."""
    m = model(cache_bits=bits, **kw)
    text = np.random.default_rng(2).integers(0, 1000, 50).tolist()
    whole = m.forward([0], [text], every=True).float()
    parts = torch.cat([m.forward([1], [text[a:b]], every=True).float() for a, b in PARTS])
    return whole, parts, m


@pytest.mark.parametrize("kw", (dict(), dict(kv_heads=4, page_size=32), dict(interleaved=True, rotary=64)))
def test_sixteen_bits_in_parts(cuda_lib, kw):
    """Different kernels multiply one row and fifty.  A dozen fp16 roundings (2^-11) lie on the way through two layers, the last of them of logits up to
    the largest; with as many again for their growth through norm and attention, 24 of them for the worst of 50000 logits and 4 for their norm."""
    whole, parts, m = both(16, **kw)
    assert (whole - parts).abs().max() <= 24 * 2.0 ** -11 * whole.abs().max()
    assert (whole - parts).norm() <= 4 * 2.0 ** -11 * whole.norm()


@pytest.mark.parametrize("kw", (dict(), dict(kv_heads=4, page_size=32)))
def test_eight_bits_in_parts_block_by_block(cuda_lib, kw):
    """The first layer's keys and values come from the same tokens' norm: the same rows but for a matmul's rounding (fp32 sums, one to fp16), which
    may move a code by a step, 2^-3 of a value, where it lies at a border.  So block by block the scales are the same, or a factor of two apart where the
    largest value lies at theirs; values differ by no more than a step, and by less than 2^-10 of the largest in all but a few."""
    _, _, m = both(8, **kw)
    (a, sa), (b, sb) = held(m, 0, 50), held(m, 1, 50)
    ratio = (sa / sb).log2()
    assert set(ratio.unique().tolist()) <= {-1.0, 0.0, 1.0} and (ratio[0] != 0).double().mean() <= 0.02
    a, b, scale = a[0], b[0], torch.maximum(sa, sb)[0]
    off = (a - b).abs()
    assert (off <= torch.maximum(a.abs(), b.abs()) * 2.0 ** -3 + 2.0 ** -9 * scale).all()
    assert (off > 2.0 ** -10 * torch.maximum(a.abs(), b.abs()) + 2.0 ** -9 * scale).double().mean() <= 0.02
