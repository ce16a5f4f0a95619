"""b200::paged_attention where q_start leaves tokens in front of the first
sequence: they belong to no sequence and get zeros, like those behind the last
one.  The output buffer holds NaN before the call."""
import pytest
import torch

import serving_reference as ref
from compiler import runtime
from compiler.runtime import cabi

pytestmark = pytest.mark.gpu
runtime.load()
BF = torch.bfloat16


@pytest.mark.parametrize("max_q", [0, 1])
@pytest.mark.parametrize("qs,ns", [([1, 1, 1], [40, 0, 333]), ([1, 300], [90, 300]), ([0, 3], [7, 3]),
                                   ([1] * 40, [20] * 40)])
@pytest.mark.parametrize("first", [1, 7, 130])
def test_tokens_in_front_of_the_first_sequence_get_zeros(first, qs, ns, max_q):
    q, kc, vc, table, q_start, kv_len = ref.paged_inputs(qs, ns, 8, 2, 64, 16, BF, pad=2)
    want = torch.ops.b200.paged_attention(q, kc, vc, table, q_start, kv_len, 0.0, 0.0, 0, max_q)
    moved = torch.cat([torch.randn_like(q[:1]).expand(first, -1, -1), q])
    out = torch.full_like(moved, float("nan"))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    cabi.paged_attention(moved, kc, vc, table, q_start + first, kv_len, out, max_q_len=max_q, status=status)
    assert status.item() == 0
    assert out[:first].eq(0).all()
    assert torch.equal(out[first:], want)


def test_sequences_without_tokens_behind_all_tokens():
    q, kc, vc, table, _, kv_len = ref.paged_inputs([1, 1], [40, 20], 8, 2, 64, 16, BF)
    out = torch.full_like(q, float("nan"))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    end = torch.full((3,), q.shape[0], dtype=torch.int32, device="cuda")
    cabi.paged_attention(q, kc, vc, table, end, kv_len, out, status=status)
    assert status.item() == 0 and out.eq(0).all()
