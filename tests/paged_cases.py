"""Plain forms, in 64 bits, of the paged KV cache and of attention over it."""
import math

import torch

# largest magnitude of an 8-bit type
LARGEST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
# the largest power of two, and the last stored value that it takes below 2^128
LAST = {torch.float8_e4m3fn: (120, 240.0), torch.int8: (122, 63.0)}


def stored(x, dtype):
    """What rows x [..., d] (bf16) stand for once a cache of ``dtype`` holds them."""
    x = x.double()
    if dtype == torch.bfloat16:
        return x
    amax = x.abs().amax(-1, keepdim=True)
    power = torch.ceil(torch.log2(amax / LARGEST[dtype]))
    step = torch.exp2(torch.where(amax > 0, power, torch.full_like(power, -100.0)).clamp_min(-100))
    y = x / step
    if dtype == torch.int8:
        y = torch.round(y)
    else:  # three bits behind the leading one, 2^-9 at the least; even in ties
        ulp = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
        y = torch.round(y / ulp) * ulp
    power, last = LAST[dtype]  # never to 2^128
    y = torch.where(step == 2.0 ** power, y.clamp(-last, last), y) * step
    return torch.where(torch.isfinite(x).all(-1, keepdim=True), y, torch.full_like(y, math.nan))


class Plain:
    """Sequences' rows as plain lists: append, read, attend."""

    def __init__(self, dtype, kv_heads, head_dim, sequences):
        self.dtype = dtype
        self.k = [torch.zeros(0, kv_heads, head_dim, dtype=torch.float64) for _ in range(sequences)]
        self.v = [x.clone() for x in self.k]

    def append(self, k, v, new):
        at = 0
        for i, n in enumerate(new):
            self.k[i] = torch.cat((self.k[i], stored(k[at:at + n], self.dtype)))
            self.v[i] = torch.cat((self.v[i], stored(v[at:at + n], self.dtype)))
            at += n

    def attend(self, q, new, scale, window=None, sinks=0, gone=()):
        """(output, bound) [rows, heads * d] of the new rows q; ``gone``: (sequence,
        first, last) positions that no row sees.  The bound is what the kernel's
        roundings come to, all in the same direction: P and the output to bf16
        (2^-8 of a value each), scores summed in fp32 (2^-24 of the sum of
        magnitudes for each of d + 8 additions and products, twice in a
        quotient), exp2 and the sums of P in fp32 (2^-20)."""
        heads, d = q.shape[1:]
        rep = heads // self.k[0].shape[1]
        out, bound, at = [], [], 0
        for i, n in enumerate(new):
            qi = q[at:at + n].double()
            at += n
            if n == 0:
                continue
            length = len(self.k[i])
            pos = torch.arange(length - n, length)[:, None]
            key = torch.arange(length)[None, :]
            seen = key <= pos
            if window is not None:
                seen &= (key > pos - window) | (key < sinks)
            for s, lo, hi in gone:
                if s == i:
                    seen &= (key < lo) | (key >= hi)
            k = self.k[i].repeat_interleave(rep, 1).permute(1, 0, 2)  # [heads, length, d]
            v = self.v[i].repeat_interleave(rep, 1).permute(1, 0, 2)
            qh = qi.permute(1, 0, 2)
            s = (torch.matmul(qh, k.transpose(1, 2)) * scale).masked_fill(~seen, -math.inf)
            some = seen.any(-1)[None, :, None]
            p = torch.where(some, torch.exp(s - torch.where(some, s.amax(-1, keepdim=True), 0.0)),
                            0.0)
            p = p / torch.where(some, p.sum(-1, keepdim=True), 1.0)
            # (a value that no row sees reaches none)
            clean = torch.where(seen.any(0)[None, :, None], v, 0.0)
            y = torch.matmul(p, clean)
            size = torch.matmul(p, clean.abs())
            dots = torch.matmul(qh.abs(), k.abs().transpose(1, 2)) * abs(scale)
            dots = dots.masked_fill(~seen, 0.0).amax(-1, keepdim=True)
            off = size * (2.0 ** -8 + 2 * (d + 8) * 2.0 ** -24 * dots + 2.0 ** -20)
            off = off + 2.0 ** -8 * (y.abs() + off)
            out.append(y.permute(1, 0, 2).reshape(n, heads * d))
            bound.append(off.permute(1, 0, 2).reshape(n, heads * d))
        return torch.cat(out), torch.cat(bound)
