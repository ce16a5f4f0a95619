"""b200::add_rms_norm_quant whose rows reach the largest magnitudes of fp32:
scales, and codes that use them, up to a maximum next to 2^128."""
import pytest
import torch

from compiler import runtime

pytestmark = pytest.mark.gpu
runtime.load()


@pytest.mark.parametrize("top", [2.0**120, 2.0**126, 1.5 * 2.0**126, 2.0**127, 1.9 * 2.0**127])
@pytest.mark.parametrize("cols,group", [(256, 0), (256, 128), (99, 0), (8200, 0), (40064, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_scales_of_the_largest_magnitudes(dtype, cols, group, top):
    """Every |sum| is 1, so the norm keeps it (eps 0) and y = +-w: the codes
    are w / scale, an e4m3 number each up to 2^-4 of itself."""
    g = torch.Generator("cuda").manual_seed(cols)
    x = torch.randint(0, 2, (3, cols), device="cuda", generator=g).mul(2).sub(1).to(dtype)
    w = torch.rand(cols, device="cuda", generator=g) * 0.98 + 0.01
    w[::64] = 1.0
    w = w * top
    q, scale, _ = torch.ops.b200.add_rms_norm_quant(x, torch.zeros_like(x), w, 0.0, group)
    want = x.double() * w.double()
    width = group or cols
    assert ((scale.double() - top / 448).abs() <= top / 448 * 1e-6).all()
    got = q.double() * scale.double().repeat_interleave(width, 1)
    assert ((got - want).abs() <= want.abs() * (2.0**-4 + 1e-4) + top / 448 * 2.0**-10).all()
