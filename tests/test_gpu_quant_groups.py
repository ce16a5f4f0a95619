"""b200::quant_groups against the formula in 64 bits.

Bounds.  y without a gate is x.  silu(g) u in fp32: the exponential errs by
(2 + 1.2 |g|) * 2^-23 relative, the division and products by 4 * 2^-23 more.
scale: two roundings of fp32, 2^-23, on top of y's.  out: half a step of e4m3 at
y / scale, which fp32 puts 2^-22 off."""
import pytest
import torch

import quant_reference as ref
from compiler import runtime

pytestmark = pytest.mark.gpu
runtime.load()
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def check(x, swiglu):
    out, scale = torch.ops.b200.quant_groups(x, swiglu)
    y = ref.silu_mul(x) if swiglu else x.double()
    err = 0.0
    if swiglu:
        gate = x.double().chunk(2, -1)[0].abs().amax().item() if x.numel() else 0.0
        err = (6 + 1.2 * gate) * 2.0**-23
    want = ref.scales(y)
    assert out.dtype == ref.E4M3 and out.shape == y.shape and scale.shape == want.shape
    assert ((scale.double() - want).abs() <= want * (err + 2.0**-22)).all()
    z = y / ref.spread(scale.double(), y.shape[-1])
    assert ((out.double() - z).abs() <= ref.code_step(z) + z.abs() * (2 * err + 2.0**-21)).all()


def make(*shape, dtype, seed=0):
    g = torch.Generator("cuda").manual_seed(seed + sum(shape))
    x = torch.randn(*shape, device="cuda", generator=g) * 2.0 ** torch.randint(-6, 4, shape[:-1] + (1,), device="cuda", generator=g)
    return x.to(dtype)


SHAPES = [(1, 128), (1, 1), (3, 7), (5, 130), (2, 1000), (64, 4096), (33, 520), (1, 40000), (300, 2056), (17, 2048), (2000, 4096),
          (1237, 136)]


@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_against_the_formula(rows, cols, dtype, swiglu):
    check(make(rows, cols * (1 + swiglu), dtype=dtype), swiglu)


@pytest.mark.parametrize("swiglu", [False, True])
def test_strides_and_leading_dims(swiglu):
    x = make(6, 5, 1024, dtype=torch.bfloat16)
    check(x, swiglu)
    check(x[..., :512], swiglu)
    check(x[..., 1:401], swiglu)      # rows that start off a 16-byte boundary
    check(x[:, ::2, :256], swiglu)    # leading dims that do not flatten
    check(x.transpose(0, 2), swiglu)  # columns apart
    check(x[0, 0], swiglu)
    check(x[:, :0], swiglu)
    check(x[..., :0], swiglu)


@pytest.mark.parametrize("cols", [256, 257])
def test_zeros_nan_and_infinity(cols):
    x = torch.zeros(6, cols, device="cuda", dtype=torch.bfloat16)
    x[1, 3] = float("nan")
    x[2, 130] = float("inf")
    x[3, 7], x[3, 8] = 3e38, 1.0
    x[4] = 1e-20
    out, scale = torch.ops.b200.quant_groups(x)
    small = torch.tensor(1e-12 / 448, dtype=torch.float32, device="cuda")
    assert (scale[0] - small).abs().max() <= small * 2.0**-22 and (out[0].float() == 0).all()
    assert scale[1, 0].isnan() and out[1, :128].float().isnan().all() and (out[1, 128:].float() == 0).all()
    assert scale[2, 1].isinf() and out[2, 130].float().isnan() and (out[2, 131:256].float() == 0).all()
    assert out[3, 7].float() == 448 and out[3, 8].float() == 0
    assert (scale[4] - small).abs().max() <= small * 2.0**-22 and (out[4].float() == 0).all()


def test_far_gates():
    """Gates whose exponential overflows or vanishes."""
    gate = torch.tensor([-200.0, -89.0, -88.0, -20.0, 0.0, 20.0, 88.0, 200.0], device="cuda").repeat(16)
    x = torch.cat([gate, torch.ones(128, device="cuda")])[None]
    out, scale = torch.ops.b200.quant_groups(x, True)
    y = ref.silu_mul(x)
    z = y / scale.double()
    assert ((out.double() - z).abs() <= ref.code_step(z) + z.abs() * 1e-4).all() and out[0, 7].float() == 448
