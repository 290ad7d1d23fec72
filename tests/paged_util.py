"""A paged key-value cache with sequences in it, and the definition of the operators over it in 64 bits, sequence by sequence."""
import math

import torch

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
UNIT = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8}            # largest relative error of one rounding


class Case:
    """Sequences with `new[b]` rows behind `past[b]` tokens.  Pages lie in a shuffled pool between others that are never used; whatever no
    token has reached, and the pages that nothing names, hold NaN, and so do the unused entries' pages of the table (they hold -1 or
    numbers far outside the pool)."""

    def __init__(self, new, past, heads, kv_heads, dim=128, page=16, dtype="fp16", seed=0, width=None, stride=0, fill=float("nan"), ragged=True):
        g = torch.Generator().manual_seed(seed)
        self.new, self.past, self.heads, self.kv, self.dim, self.page, self.dtype = list(new), list(past), heads, kv_heads, dim, page, dtype
        self.length = [max(a + b, 0) for a, b in zip(new, past)]
        T = DTYPES[dtype]
        used = [-(-n // page) for n in self.length]
        pool = sum(used) + 3
        order = torch.randperm(pool, generator=g)
        width = width or max(used + [1]) + 1
        table = torch.full((len(new), width), -1, dtype=torch.int32)
        table[:, -1] = 1 << 30
        at = 0
        # one storage for both, a page stride larger than a page where `stride` says so
        whole = kv_heads * page * dim
        flat = torch.full((pool, 2 * whole + stride), fill, dtype=T)
        k, v = (flat[:, i * whole:(i + 1) * whole].view(pool, kv_heads, page, dim) for i in range(2))
        self.keys, self.values = [], []
        for b, n in enumerate(used):
            table[b, :n] = order[at:at + n].int()
            kk, vv = (torch.randn((kv_heads, self.length[b], dim), generator=g).to(T) for _ in "kv")
            for i in range(n):
                part = slice(i * page, min((i + 1) * page, self.length[b]))
                k[order[at + i], :, :part.stop - part.start] = kk[:, part]
                v[order[at + i], :, :part.stop - part.start] = vv[:, part]
            self.keys.append(kk)
            self.values.append(vv)
            at += n
        self.flat = flat.cuda()
        self.k, self.v = (self.flat[:, i * whole:(i + 1) * whole].view(pool, kv_heads, page, dim) for i in range(2))
        self.table, self.lengths = table.cuda(), torch.tensor(self.length, dtype=torch.int32).cuda()
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        self.starts_list, self.tokens = starts, starts[-1]
        self.starts = torch.tensor(starts, dtype=torch.int32).cuda() if ragged else None
        self.q = torch.randn((self.tokens, heads, dim), generator=g).to(T).cuda()

    def args(self):
        return self.k, self.v, self.table, self.lengths

    def visible(self, b, causal=True, window=0, prefix=None):
        """[rows, keys] of sequence b."""
        i = torch.arange(self.past[b], self.past[b] + self.new[b])[:, None]
        j = torch.arange(self.length[b])[None]
        if not causal:
            see = torch.ones((i.shape[0], j.shape[1]), dtype=torch.bool)
        else:
            see = j <= i
            if window:
                see &= i - j < window
            if prefix is not None:
                see |= j < prefix[b]
        return see & (i >= 0), (i - j).abs()

    def reference(self, scale=None, causal=True, window=0, cap=0.0, slopes=None, prefix=None, q=None):
        """(result, bound): in 64 bits, and how far a kernel may be off.  The bound: one rounding u of the result, one of each weight
        (u of its size, in fp16 at least half the smallest subnormal, 2^-25 of the largest weight), and fp32 sums of `dim` products,
        2^-23 sqrt(dim) |q||k| in a score (four times what is usual), plus a few fp32 steps of the score itself and of exp and tanh."""
        q = (self.q if q is None else q).double().cpu()
        group, u = self.heads // self.kv, UNIT[self.dtype]
        scale = self.dim ** -0.5 if scale is None else scale
        out, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
        for b in range(len(self.new)):
            if self.length[b] == 0 or self.new[b] == 0:
                continue
            see, distance = self.visible(b, causal, window, prefix)
            rows = slice(self.starts_list[b], self.starts_list[b + 1])
            for h in range(self.heads):
                k, v = self.keys[b][h // group].double(), self.values[b][h // group].double()
                hidden = ~see.any(dim=0)
                v = v.masked_fill(hidden[:, None], 0.0)         # what no row sees does not exist
                k = k.masked_fill(hidden[:, None], 0.0)
                x = q[rows, h] @ k.T * scale
                slack = 2.0 ** -23 * math.sqrt(self.dim) * abs(scale) * q[rows, h].norm(dim=1)[:, None] * k.norm(dim=1)[None]
                if cap:
                    x = cap * torch.tanh(x / cap)
                    slack = slack + 2.0 ** -20 * cap
                if slopes is not None:
                    x = x - float(slopes[h]) * distance
                slack = slack + 2.0 ** -21 * (x.abs() + 1)
                x = x.masked_fill(~see, -math.inf)
                top = x.amax(dim=1, keepdim=True).clamp(min=-1e300)
                w = torch.exp(x - top)
                total = w.sum(dim=1, keepdim=True).clamp(min=1e-300)
                p = w / total
                o = p @ v
                out[rows, h] = o
                slack = torch.where(see, slack, 0.0).amax(dim=1, keepdim=True)
                bound[rows, h] = u * o.abs() + (u + 2 * slack) * (p @ v.abs()) + 2.0 ** -25 / total * (see.double() @ v.abs()) * (self.dtype == "fp16") + 2.0 ** -24
        return out, bound


def assert_within(got, reference, what=""):
    ref, bound = reference
    got = got.double().cpu()
    assert torch.isfinite(got).all(), f"{what}: non-finite values"
    off = (got - ref).abs()
    worst = int((off - bound).argmax())
    assert (off <= bound).all(), f"{what}: |{got.flatten()[worst]} - {ref.flatten()[worst]}| > {bound.flatten()[worst]:.3e} at {worst}"
