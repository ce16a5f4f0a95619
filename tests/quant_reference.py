"""Plain 64-bit forms of the 8-bit operators, and inputs for their tests."""
from __future__ import annotations

import torch

E4M3 = torch.float8_e4m3fn
MAX, MIN_AMAX = 448.0, 1e-12


def groups(y):
    """[..., cols] as a list of its groups of 128 columns, the last one what is left."""
    return y.split(128, -1)


def scales(y):
    """max(max |y|, 1e-12) / 448 of each group of 128 columns, in 64 bits."""
    if y.shape[-1] == 0:
        return y.double()
    return torch.stack([g.abs().amax(-1) for g in groups(y.double())], -1).clamp_min(MIN_AMAX) / MAX


def spread(scale, cols):
    """[..., groups] over the columns that they scale."""
    return scale.repeat_interleave(128, -1)[..., :cols]


def silu_mul(x):
    gate, up = x.double().chunk(2, -1)
    return gate / (1 + torch.exp(-gate)) * up


def code_step(y):
    """Half a step of e4m3 around y: 2^-4 relative, 2^-10 below the smallest normal number 2^-6."""
    return torch.maximum(y.abs() * 2.0**-4, torch.full_like(y, 2.0**-10))


def random_codes(rows, cols, g, spread_exp=4):
    """e4m3 codes of every sign and of many exponents, and positive scales."""
    x = torch.randn(rows, cols, device="cuda", generator=g) * 2.0 ** torch.randint(-spread_exp, spread_exp, (rows, cols),
                                                                                device="cuda", generator=g)
    return x.clamp(-MAX, MAX).to(E4M3)


def random_scales(*shape, g):
    return 2.0 ** (torch.rand(*shape, device="cuda", generator=g) * 8 - 8)


def scaled_mm(a, b, a_scale, b_scale):
    """(a @ b with the scales, sum of the products' magnitudes) in 64 bits."""
    k, n = b.shape
    da = a.double() * spread(a_scale.double(), k)
    db = b.double() * spread(spread(b_scale.double(), n).t(), k).t()
    return da @ db, da.abs() @ db.abs()
