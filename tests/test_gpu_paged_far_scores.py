"""b200::paged_attention where one key outweighs all others by many orders of
magnitude and its value is zero, so that the output is the others' alone
(as behind a first key that draws the softmax to itself).

The bound is serving_reference.attention_close's: half a step of the type for
each probability.  It supposes probabilities that the type holds as normal
numbers.  f16 ones are scaled by 2^15 (row kernel) and 2^12 (tile kernel), so
they are normal from 2^-14 - 12 = 2^-26 of the row's maximum on, 18 nats: the
distances here are no larger."""
import pytest
import torch

import serving_reference as ref
from compiler import runtime

pytestmark = pytest.mark.gpu
runtime.load()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m", [1, 5, 100])  # rows, two row blocks, tiles
@pytest.mark.parametrize("sink", [0, 130])
@pytest.mark.parametrize("nats", [9.0, 13.0, 16.0, 18.0])
@pytest.mark.parametrize("D", [64, 128])
def test_a_key_far_above_the_others(D, nats, sink, m, dtype):
    n = 400
    q, kc, vc, table, q_start, kv_len = ref.paged_inputs([m, m], [n, 290], 8, 2, D, 16, dtype)
    q = torch.zeros_like(q)
    q[..., 0] = 8.0
    q[..., 1] = 1.0
    kc[..., 0] = 0.0
    kc[table[:, sink // 16].long(), sink % 16, :, 0] = nats * D**0.5 / 8.0
    vc += 100.0
    vc[table[:, sink // 16].long(), sink % 16] = 0.0
    args = q, kc, vc, table, q_start, kv_len
    want, size = ref.paged_attention(*args, ref.default_scale(D))
    ref.attention_close(torch.ops.b200.paged_attention(*args), want, size, dtype)


@pytest.mark.parametrize("m", [1, 64])
def test_a_first_key_far_above_a_long_tail(m):
    """Thousands of keys that share a warp's run with the first one."""
    dtype, D, n, seqs = torch.float16, 64, 5000, 160 if m == 1 else 1
    q, kc, vc, table, q_start, kv_len = ref.paged_inputs([m] * seqs, [n] * seqs, 8, 1, D, 64, dtype)
    q = torch.zeros_like(q)
    q[..., 0] = 8.0
    kc[..., 0] = 0.0
    kc[table[:, 0].long(), 0, :, 0] = 17.0
    vc += 10.0
    vc[table[:, 0].long(), 0] = 0.0
    args = q, kc, vc, table, q_start, kv_len
    want, size = ref.paged_attention(*args, ref.default_scale(D))
    ref.attention_close(torch.ops.b200.paged_attention(*args), want, size, dtype)
