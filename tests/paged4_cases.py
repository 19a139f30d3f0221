"""Plain forms, in 64 bits, of the paged KV cache in 4 bits."""
import math

import torch

from paged_cases import Plain
from test_gpu_paged import Run

E2M1 = torch.float4_e2m1fn_x2


def stored(x, group):
    """What rows x [..., d] (bf16) stand for once a cache of 4 bits holds them, a power of
    two for `group` of their dims."""
    x = x.double().unflatten(-1, (-1, group))
    amax = x.abs().amax(-1, keepdim=True)
    power = torch.ceil(torch.log2(amax / 7.0))
    step = torch.exp2(torch.where(amax > 0, power, torch.full_like(power, -100.0))
                      .clamp(-100, 125))
    z = x / step
    # one bit behind the leading one, halves below 1, 6 at the most; even in ties
    ulp = torch.exp2(torch.floor(torch.log2(z.abs().clamp(1.0, 6.0))) - 1)
    y = (torch.round(z / ulp) * ulp).clamp(-6.0, 6.0) * step
    y = torch.where(torch.isfinite(x).all(-1, keepdim=True), y, torch.full_like(y, math.nan))
    return y.flatten(-2)


class Plain4(Plain):
    def append(self, k, v, new):
        at = 0
        for i, n in enumerate(new):
            self.k[i] = torch.cat((self.k[i], stored(k[at:at + n], 32)))
            self.v[i] = torch.cat((self.v[i], stored(v[at:at + n], v.shape[-1])))
            at += n


class Run4(Run):
    """Sequences in a cache of 4 bits and in the plain form."""

    def __init__(self, kv_heads, d, page, steps, seed=0):
        super().__init__(E2M1, kv_heads, d, page, steps, seed)
        self.plain = Plain4(torch.bfloat16, kv_heads, d, len(steps[0]))
