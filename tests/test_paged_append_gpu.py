"""Rotary positions and the append to the pages against complex multiplication in 64 bits."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from paged_util import UNIT, Case
from relax_b200 import B200Error, ops

pytestmark = pytest.mark.gpu


def tables(positions, rotary):
    angle = np.arange(positions)[:, None] * 10000.0 ** (-np.arange(rotary // 2) * 2.0 / rotary)
    return (torch.from_numpy(f(angle).astype(np.float32)).cuda() for f in (np.cos, np.sin))


def check(c, rotary, interleaved, positions=None, pad=0):
    rng = torch.Generator().manual_seed(5)
    width = (c.heads + 2 * c.kv) * c.dim
    qkv = torch.randn((c.tokens, width + pad), generator=rng).to(c.q.dtype).cuda()[:, :width]
    cos, sin = tables(max(c.length + [1]) + 3, rotary)
    before = c.flat.clone()
    q = ops.paged_rope_append(qkv, cos, sin, *c.args(), starts=c.starts, interleaved=interleaved,
                              positions=None if positions is None else torch.tensor(positions, dtype=torch.int32).cuda())
    torch.cuda.synchronize()
    rows = qkv.double().cpu().numpy().reshape(c.tokens, -1, c.dim)
    ct, st = cos.double().cpu().numpy(), sin.double().cpu().numpy()
    half, u = rotary // 2, UNIT[c.dtype]
    after = before.clone()
    k, v = (after[:, i * c.kv * c.page * c.dim:(i + 1) * c.kv * c.page * c.dim].view(c.k.shape) for i in range(2))
    for b in range(len(c.new)):
        for i in range(c.new[b]):
            row, at = c.starts_list[b] + i, c.past[b] + i
            if at < 0:
                assert (q[row] == 0).all()
                continue
            x = rows[row].copy()
            turn = ct[at] + 1j * st[at] if positions is None else ct[positions[row]] + 1j * st[positions[row]]
            part = x[: c.heads + c.kv, :rotary]
            a, d = (part[:, 0::2], part[:, 1::2]) if interleaved else (part[:, :half], part[:, half:])
            z = (a + 1j * d) * turn
            size = np.abs(a) + np.abs(d)              # fp32: two products and a sum, each 2^-24 of at most this
            y = np.empty_like(part)
            if interleaved:
                y[:, 0::2], y[:, 1::2] = z.real, z.imag
            else:
                y[:, :half], y[:, half:] = z.real, z.imag
            slack = np.repeat(size, 2, axis=1) if interleaved else np.concatenate([size, size], axis=1)
            bound = u * np.abs(y) + 3 * 2.0 ** -24 * slack + (2.0 ** -25 if c.dtype == "fp16" else 0)
            page, slot = int(c.table[b, at // c.page]), at % c.page
            got_k = c.k[page, :, slot].double().cpu().numpy()
            got = np.concatenate([q[row].double().cpu().numpy(), got_k])
            assert (np.abs(got[:, :rotary] - y) <= bound).all()
            assert (got[:, rotary:] == x[: c.heads + c.kv, rotary:]).all()
            k[page, :, slot] = c.k[page, :, slot]
            v[page, :, slot] = qkv[row, (c.heads + c.kv) * c.dim:].view(c.kv, c.dim)
    # everything else is as it was, and v is there to the bit
    assert torch.equal(c.flat.view(torch.int16), after.view(torch.int16))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary", [(128, 128), (128, 64), (128, 48), (128, 16), (64, 64), (64, 32), (64, 16)])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_layouts(cuda_lib, interleaved, dim, rotary, dtype):
    check(Case([3, 1, 20], [0, 40, 29], 6, 2, dim, 32, dtype, stride=8), rotary, interleaved, pad=24)


@pytest.mark.parametrize("heads,kv,page", [(1, 1, 16), (32, 32, 16), (40, 8, 128), (65, 1, 64), (7, 7, 16)])
def test_one_token_each(cuda_lib, heads, kv, page):
    n = [1, 15, 16, 17, 33, 100]
    check(Case([1] * len(n), [x - 1 for x in n], heads, kv, 128, page, ragged=False), 128, False)


def test_positions_of_their_own_and_rows_without_a_place(cuda_lib):
    check(Case([4, 2, 0, 5], [9, -1, 3, -7], 4, 2), 128, False)
    check(Case([4, 2, 0, 5], [9, 1, 3, 0], 4, 2), 64, True, positions=[0, 3, 1, 2, 9, 9, 0, 1, 12, 4, 5])


def test_many_sequences(cuda_lib):
    check(Case([i % 4 for i in range(70)], [i * 7 % 50 for i in range(70)], 2, 1, 64, 16), 64, False)


def test_refusals(cuda_lib):
    c = Case([1, 1], [3, 4], 4, 2, ragged=False)
    qkv = torch.zeros((2, 8 * 128), dtype=torch.float16, device="cuda")
    cos, sin = tables(10, 128)

    def call(qkv=qkv, cos=cos, sin=sin, k=c.k, v=c.v, table=c.table, lengths=c.lengths, **kw):
        return ops.paged_rope_append(qkv, cos, sin, k, v, table, lengths, **kw)

    call()
    for bad in (dict(qkv=qkv.float()), dict(qkv=qkv[:, :4 * 128]), dict(qkv=qkv[:, :1000]), dict(cos=cos.half()), dict(sin=sin[:5]),
                dict(cos=cos[:, :20].contiguous(), sin=sin[:, :20].contiguous()), dict(lengths=c.lengths[:1]), dict(k=c.k.float(), v=c.v.float()),
                dict(positions=torch.zeros(3, dtype=torch.int32).cuda()), dict(out=qkv), dict(qkv=qkv.cpu()), dict(cos=cos[:0], sin=sin[:0]),
                dict(qkv=torch.zeros((2, 8 * 128 + 4), dtype=torch.float16, device="cuda")[:, :8 * 128])):
        with pytest.raises((ValueError, B200Error)):
            call(**bad)
    assert call(qkv=qkv[:0], table=c.table[:0], lengths=c.lengths[:0]).shape == (0, 4, 128)
