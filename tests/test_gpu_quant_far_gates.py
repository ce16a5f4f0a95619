"""b200::quant_groups with gates far below zero beside very large values.

e^-|g| is at least 2^-133 for |g| <= 92, where fp32's smallest step, 2^-149, is 2^-16 of
it; two roundings to it (the exponential, its product with 1 / (1 + e^-|g|)) are half
a step each, the exponential's own error (2 + 1.2 |g|) 2^-23 = 1.4e-5 and the others below
2^-21: y is within 2^-16 + 1.5e-5 < 2^-15 of itself, a group's scale too."""
import pytest
import torch

import quant_reference as ref
from compiler import runtime

pytestmark = pytest.mark.gpu
runtime.load()


@pytest.mark.parametrize("off", [0, 1])  # the vector kernel and the other
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_far_gates_and_large_values(dtype, off):
    gate = -torch.linspace(80, 92, 25, device="cuda")[:, None].expand(25, 128)
    up = 2.0 ** torch.randint(110, 128, (25, 128), device="cuda", generator=torch.Generator("cuda").manual_seed(0)).float()
    x = torch.cat([gate, up], 1).to(dtype)
    x = torch.nn.functional.pad(x, (off, 0))[:, off:]
    out, scale = torch.ops.b200.quant_groups(x, True)
    y = ref.silu_mul(x)
    want = ref.scales(y)
    assert ((scale.double() - want).abs() <= want * 2.0**-15).all()
    z = y / scale.double()
    assert ((out.double() - z).abs() <= ref.code_step(z) + z.abs() * 2.0**-14).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_infinite_gates(dtype):
    inf = float("inf")
    x = torch.ones(3, 256, device="cuda")
    x[0, 5], x[1, 5], x[2, 5] = inf, -inf, float("nan")
    out, scale = torch.ops.b200.quant_groups(x.to(dtype), True)
    assert scale[0].isinf().all() and out[0, 5].float().isnan() and out[0, 6].float() == 0
    assert scale[1:].isnan().all() and out[1:].float().isnan().all()
