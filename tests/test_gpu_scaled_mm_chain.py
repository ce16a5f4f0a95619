"""b200::scaled_mm in chains without a pause: CTA pairs that leave while the next
call's CTAs, of any tile, take their shared memory and tensor memory."""
import pytest
import torch

from compiler import runtime
from test_gpu_scaled_mm import check, make

pytestmark = pytest.mark.gpu
runtime.load()
BF = torch.bfloat16


def test_wide_products_in_a_row():
    """The bits of every call are those of the call alone; k of one block and of many, so that pairs
    leave right behind their last product."""
    args = [make(m, k, n) for m, k, n in ((2048, 128, 2560), (600, 256, 4000), (7, 1024, 4096), (2000, 1152, 2000), (100, 128, 8192))]
    alone = []
    for a in args:
        alone.append(torch.ops.b200.scaled_mm(*a, BF))
        torch.cuda.synchronize()
        check(alone[-1], *a)
    outs = [[torch.ops.b200.scaled_mm(*a, BF) for a in args] for _ in range(40)]
    torch.cuda.synchronize()
    for row in outs:
        for got, want in zip(row, alone):
            assert torch.equal(got, want)
    assert runtime.gemm_status() == 0
