"""b200::paged_attention with caps of every size, near the scores and far
above them, on both kernels.

The bound is serving_reference.attention_close's: fp32 scores below 64 that
are off by at most 2.4e-4.  The cap adds at most 5e-5: up to a cap of 100 an
error of 3.6e-7 of the cap, above it one of less than 7e-7 of the score.  Where
scores go up to 64 heads are of 64, half of those 2.4e-4."""
import pytest
import torch

import serving_reference as ref
from compiler import runtime

pytestmark = pytest.mark.gpu
runtime.load()


@pytest.mark.parametrize("cap", [3.0, 50.0, 100.0, 100.5, 1e3, 1e4, 1e5, 1e7, 1e20, 1e38])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m", [1, 5, 150])  # rows, two row blocks, tiles
@pytest.mark.parametrize("D", [64, 128])
def test_caps(D, m, dtype, cap):
    args = ref.paged_inputs([m, 1], [200, 90], 8, 2, D, 16, dtype)
    out = torch.ops.b200.paged_attention(*args, 0.0, cap)
    want, size = ref.paged_attention(*args, ref.default_scale(D), cap)
    ref.attention_close(out, want, size, dtype)


@pytest.mark.parametrize("cap", [10.0, 20.0, 40.0, 100.0, 101.0])
@pytest.mark.parametrize("m", [1, 150])
def test_scores_that_reach_the_cap(m, cap):
    """Scores of up to about 40: with the larger caps on both sides of 0.35 of it."""
    args = ref.paged_inputs([m, 1], [200, 90], 8, 2, 64, 16, torch.bfloat16)
    out = torch.ops.b200.paged_attention(*args, 0.5, cap)
    want, size = ref.paged_attention(*args, 0.5, cap)
    ref.attention_close(out, want, size, torch.bfloat16)
