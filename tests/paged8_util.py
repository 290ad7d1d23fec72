"""Pages of 8 bits with scales, and the definition of what is done with them in 64 bits."""
import math

import torch

import paged_util
from paged_util import DTYPES, UNIT

E4M3 = torch.float8_e4m3fn
LEAST, MOST = -24, 7                             # powers of two that a scale may be


def power_for(most):
    """The exponent of the smallest power of two by which values up to `most` are at most 448."""
    if not most > 0:
        return LEAST
    part, e = math.frexp(most)                   # most / 448 = part 2^e / (0.875 * 2^9)
    return min(max(e - 9 + (part > 0.875), LEAST), MOST)


def to_e4m3(x):
    """To the nearest number of the format (ties to even), in 64 bits; at most 448 in size."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


class Case8(paged_util.Case):
    """As Case, its keys and values in 8 bits: `k8`, `v8` [pages, kv, page, dim], `k_scales`, `v_scales`; keys and values are what the codes stand for.
    Blocks' sizes differ by factors of `spread`.  What no token has reached holds NaN, codes and scales."""

    def __init__(self, *args, spread=4.0, **kw):
        super().__init__(*args, **kw)
        g = torch.Generator().manual_seed(kw.get("seed", 0) + 1000)
        pool, page = self.k.shape[0], self.page
        table = self.table.cpu()
        for name, held in (("k", self.keys), ("v", self.values)):
            codes = torch.full((pool, self.kv, page, self.dim), 0x7f, dtype=torch.uint8)
            scales = torch.full((pool, self.kv, page // 16), float("nan"), dtype=torch.float16)
            for b, n in enumerate(self.length):
                whole = torch.zeros((self.kv, -(-n // 16) * 16, self.dim), dtype=torch.float64)
                for i in range(0, n, 16):
                    part = held[b][:, i:i + 16].double() * (spread ** torch.randn((self.kv, 1, 1), generator=g, dtype=torch.float64))
                    for h in range(self.kv):
                        scale = 2.0 ** power_for(float(part[h].abs().max()))
                        code = to_e4m3(part[h] / scale)
                        at = int(table[b, i // page])
                        codes[at, h, i % page:i % page + part.shape[1]] = code.to(E4M3).view(torch.uint8)
                        scales[at, h, i % page // 16] = scale
                        whole[h, i:i + part.shape[1]] = code * scale
                held[b] = whole[:, :n]
            setattr(self, name + "8", codes.view(E4M3).cuda())
            setattr(self, name + "_scales", scales.cuda())

    def args(self):
        return self.k8, self.v8, self.table, self.lengths

    def scales(self):
        return dict(k_scales=self.k_scales, v_scales=self.v_scales)

    def reference(self, scale=None, causal=True, window=0, cap=0.0, slopes=None, prefix=None, q=None):
        """As Case.reference.  The bound there counts one rounding of the result and of each weight by the rows' type and fp32 sums; weights are
        rounded to fp16 here, so bf16 rows get no more than that.  On top of it: what lies below fp16's normal numbers, 2^-25 of the largest weight
        times value, for every value's code (448 at most, of a block whose scale is the largest of all), and 2^-25 of a key or a value itself."""
        out, bound = super().reference(scale, causal, window, cap, slopes, prefix, q)
        q = (self.q if q is None else q).double().cpu()
        factor = self.dim ** -0.5 if scale is None else abs(scale)
        for b, n in enumerate(self.length):
            rows = slice(self.starts_list[b], self.starts_list[b + 1])
            if n == 0 or rows.start == rows.stop:
                continue
            for h in range(self.heads):
                v = self.values[b][h // (self.heads // self.kv)].abs()
                far = 2.0 ** -25 * factor * q[rows, h].abs().sum(dim=1, keepdim=True)          # of a score, by keys that small
                bound[rows, h] += 2 * far * v.amax() + 2.0 ** -25 * (n + 1) * v.amax() * (448 / 256) + 2.0 ** -25
        return out, bound
