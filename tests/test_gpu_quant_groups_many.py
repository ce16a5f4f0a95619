"""b200::quant_groups of prompt-sized inputs, whose threads take four groups each
(from 2048 groups an SM on): groups that end inside a row's last 128 columns, and
counts that leave the last CTA some of its 64.  Bounds: test_gpu_quant_groups.check,
a part of the rows at a time."""
import pytest
import torch

import quant_reference as ref
from compiler import runtime
from compiler.runtime import cabi
from test_gpu_quant_groups import make

pytestmark = pytest.mark.gpu
runtime.load()


@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,cols", [(16385, 2440), (40001, 1000), (310001, 128), (305003, 8)])
def test_four_groups_a_thread(rows, cols, dtype, swiglu):
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    groups = rows * -(-cols // 128)
    assert groups >= 2048 * sms and groups % 64
    x = make(rows, cols * (1 + swiglu), dtype=dtype)
    gate = x[:, :cols].abs().amax().item() if swiglu else 0.0
    err = (6 + 1.2 * gate) * 2.0**-23 if swiglu else 0.0
    out, scale = torch.ops.b200.quant_groups(x, swiglu)
    assert out.shape == (rows, cols) and scale.shape == (rows, -(-cols // 128))
    for part, codes, s in zip(x.split(8192), out.split(8192), scale.split(8192)):
        y = ref.silu_mul(part) if swiglu else part.double()
        want = ref.scales(y)
        assert ((s.double() - want).abs() <= want * (err + 2.0**-22)).all()
        z = y / ref.spread(s.double(), cols)
        assert ((codes.double() - z).abs() <= ref.code_step(z) + z.abs() * (2 * err + 2.0**-21)).all()


def test_rows_and_groups_behind_the_last_one():
    """Of a strided input, into the allocator's own memory: what lies behind is left as it was."""
    rows, cols = 33333, 1160
    x = make(rows, cols + 24, dtype=torch.bfloat16)[:, :cols]
    out, scale = torch.ops.b200.quant_groups(x)
    again, scale2 = torch.ops.b200.quant_groups(x.contiguous())
    assert torch.equal(out.view(torch.uint8), again.view(torch.uint8)) and torch.equal(scale, scale2)
    n, g = rows * cols, rows * -(-cols // 128)
    wide, wide_s = torch.full((n + 512,), 9, dtype=torch.uint8, device="cuda"), torch.full((g + 64,), 9.0, device="cuda")
    cabi.quant_groups(x, wide[:n].view(rows, cols), wide_s[:g].view(rows, -1))
    assert torch.equal(wide[:n], out.view(torch.uint8).flatten()) and torch.equal(wide_s[:g], scale.flatten())
    assert (wide[n:] == 9).all() and (wide_s[g:] == 9).all()
