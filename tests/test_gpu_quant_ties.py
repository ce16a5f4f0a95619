"""Codes of 16-bit values, bit for bit: y / scale lies half way between two e4m3
numbers often when y and a group's largest value have 8 or 11 bits (3 codes in
10000 of normal bf16 values), and the code is the even one.

y * 448 / top in 64 bits is exact where it is half way (at most 5 bits), and
elsewhere at least 1 / (31 * 2^11) of itself away, relative, so its conversion by
way of fp32 (2^-24) is the formula's code and no tolerance is needed."""
import pytest
import torch

import quant_reference as ref
from compiler import runtime

pytestmark = pytest.mark.gpu
runtime.load()
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def exact(y):
    """The codes of y's rows, one scale each."""
    y = y.double()
    return (y * ref.MAX / y.abs().amax(-1, keepdim=True).clamp_min(ref.MIN_AMAX)).float().to(ref.E4M3)


def same(got, want):
    assert torch.equal(got.view(torch.uint8), want.view(torch.uint8))


def randn(*shape, dtype, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


@pytest.mark.parametrize("as_f32", [False, True])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rows,cols", [(64, 4096), (3000, 1024), (5, 130), (200, 777)])
def test_quant_groups(rows, cols, dtype, as_f32):
    x = randn(rows, cols, dtype=dtype, seed=rows + cols)
    out, _ = torch.ops.b200.quant_groups(x.float() if as_f32 else x)
    for got, part in zip(out.split(128, 1), x.split(128, 1)):
        same(got, exact(part))


def test_quant_groups_half_way():
    """Values t a / 3584, t odd, of every bf16 mantissa a: half way wherever they need no rounding."""
    a = (128 + torch.arange(128, device="cuda")).to(BF)
    x = torch.zeros(128, 128, device="cuda", dtype=BF)
    x[:, 0] = a
    for i, t in enumerate(torch.arange(17, 512, 2).tolist()[:100]):
        x[:, 1 + i] = (a.double() * t / 448 / 2.0**3).to(BF)
    out, _ = torch.ops.b200.quant_groups(x)
    same(out, exact(x))
    x = torch.nn.functional.pad(x, (1, 0))[:, 1:]  # off a 16-byte boundary
    out, _ = torch.ops.b200.quant_groups(x)
    same(out, exact(x))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("tokens", [3, 5000])
@pytest.mark.parametrize("dim", [64, 128, 80, 48])
def test_appended_rows(dim, tokens, dtype):
    """Values, and keys that are not turned."""
    q, k, v = (randn(tokens, h, dim, dtype=dtype, seed=i) for i, h in enumerate((8, 3, 3)))
    caches = [torch.zeros(tokens, 1, 3, dim, device="cuda", dtype=torch.uint8).view(ref.E4M3) for _ in range(2)]
    scales = [torch.zeros(tokens, 1, 3, device="cuda") for _ in range(2)]
    none, at = torch.ones(1, 0, device="cuda"), torch.arange(tokens, device="cuda")
    torch.ops.b200.rope_append_quant(q, k, v, none, none, at * 0, at, *caches, *scales)
    same(caches[0][:, 0], exact(k))
    same(caches[1][:, 0], exact(v))
