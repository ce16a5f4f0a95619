"""The tile kernels of the paged attentions when a wait runs out in the middle of a
list of units: CTAs with several portions, whose loaders are blocks and queries
ahead of the products that stopped.  Everything in flight is waited for, the call
is reported, and the next one is right."""
import pytest
import torch

import quant_cache as qc
import serving_reference as ref
from compiler import runtime
from compiler.runtime import cabi

pytestmark = pytest.mark.gpu
runtime.load()
BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("page", [16, 12])  # TMA boxes and row by row
@pytest.mark.parametrize("queries", [130, 256])  # portions of 3 and of 4 key blocks
@pytest.mark.parametrize("D,dtype", [(64, BF), (128, HF)])
@pytest.mark.parametrize("e4m3", [False, True])
def test_a_stall_with_portions_ahead(e4m3, D, dtype, queries, page):
    seqs = 150
    inputs = (qc if e4m3 else ref).paged_inputs([queries] * seqs, [queries] * seqs, 4, 4, D, page, dtype)
    call = cabi.paged_attention_quant if e4m3 else cabi.paged_attention
    out, status = torch.zeros_like(inputs[0]), torch.zeros(1, dtype=torch.int32, device="cuda")
    for _ in range(3):
        call(*inputs, out, status=status, timeout_ns=20_000_000, test_flags=cabi.PAGED_TEST_WITHHOLD_SCORES)
        torch.cuda.synchronize()
        assert status.item() == 6
        status.zero_()
    call(*inputs, out, status=status)
    torch.cuda.synchronize()
    assert status.item() == 0
    again = torch.empty_like(out)
    call(*inputs, again, status=status)
    assert torch.equal(out, again)
    # the last two sequences against the formula
    q, *caches, table, starts, lens = inputs
    some = (q[-2 * queries:], *caches, table[-2:], starts[:3], lens[-2:])
    if e4m3:
        qc.attention_close(out[-2 * queries:], some, ref.default_scale(D))
    else:
        ref.attention_close(out[-2 * queries:], *ref.paged_attention(*some, ref.default_scale(D)), dtype)
