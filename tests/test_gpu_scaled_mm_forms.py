"""b200::scaled_mm: forms of the output's last columns and of the persistent loop, each
against the formula in 64 bits (bound: test_gpu_scaled_mm.check)."""
import pytest
import torch

from compiler import runtime
from compiler.runtime import cabi
from test_gpu_scaled_mm import check, make

pytestmark = pytest.mark.gpu
runtime.load()
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def forced(m, k, n, dtype, tile, split=0):
    a, b, sa, sb = make(m, k, n)
    out = torch.full((m + 2, n), 7.0, device="cuda", dtype=dtype)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    cabi.scaled_mm(a, b, sa, sb, out[:m], tile=tile, split=split, status=status)
    assert status.item() == 0
    check(out[:m], a, b, sa, sb)
    assert (out[m:] == 7.0).all()  # nothing behind the last row


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 2, 3, 4, 66, 67, 68, 129, 195, 258, 1025, 1026, 1027, 1028, 1090, 1091, 1154, 1219])
@pytest.mark.parametrize("m,k", [(300, 128), (513, 896)])
def test_wide_tiles_of_rows_of_every_alignment(m, k, n, dtype):
    """Columns that end inside each 64 of a warp, in stores of two, four and eight bytes and by TMA."""
    forced(m, k, n, dtype, 1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [4096, 4097, 4098, 4100])
def test_wide_tiles_by_the_library_s_choice(n, dtype):
    a, b, sa, sb = make(1024, 256, n)
    check(torch.ops.b200.scaled_mm(a, b, sa, sb, dtype), a, b, sa, sb)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", [128, 384, 1152, 2176])  # 1, 3, 9, 17 blocks: both issuers and chunks of scales change places
@pytest.mark.parametrize("tile,m", [(16, 40), (32, 100), (64, 100), (64, 130), (128, 200)])
def test_several_tiles_a_cta(tile, m, k, dtype):
    """157 tiles of columns by 2 to 4 of rows on 296 CTAs (128 rows: 148)."""
    forced(m, k, 20000, dtype, tile, 1)


@pytest.mark.parametrize("m", [30, 60, 100, 128])
def test_several_tiles_a_cta_by_the_library_s_choice(m):
    a, b, sa, sb = make(m, 1152, 50000)
    check(torch.ops.b200.scaled_mm(a, b, sa, sb, torch.bfloat16), a, b, sa, sb)
