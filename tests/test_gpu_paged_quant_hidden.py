"""b200::paged_attention_quant: values that a query does not see, and values that it
gives no weight, leave its output as it is, however large they are beside the others.

Bound: serving_reference.attention_close, on what codes and scales stand for, for
both types (weights are rounded to f16, codes enter as they are)."""
import pytest
import torch

import quant_cache as qc
import serving_reference as ref
from compiler import runtime

pytestmark = pytest.mark.gpu
runtime.load()
BF, HF = torch.bfloat16, torch.float16
op = torch.ops.b200.paged_attention_quant


def close(out, x, softcap=0.0, window=0):
    q = x[0]
    want, size = qc.attend(x, ref.default_scale(q.shape[2]), softcap, window)
    ref.attention_close(out, want, size, q.dtype)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("m", [3, 20, 150])  # rows, two row blocks, tiles
@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("up", [20, 40, 100, -60])
def test_large_values_of_hidden_keys(up, cap, m, D, dtype):
    """The last key, and one in the middle of the queries, 2^up times the others."""
    n = 260
    q, k8, v8, ks, vs, table, q_start, kv_len = qc.paged_inputs([m], [n], 8, 2, D, 16, dtype)
    clean = op(q, k8, v8, ks, vs, table, q_start, kv_len, 0.0, cap)
    close(clean, (q, k8, v8, ks, vs, table, q_start, kv_len), cap)
    far = vs.clone()
    keys = [n - 1, n - 1 - m // 2]
    for key in keys:
        far[table[0, key // 16].long(), key % 16] *= 2.0**up
    out = op(q, k8, v8, ks, far, table, q_start, kv_len, 0.0, cap)
    hidden = torch.arange(n - m, n, device="cuda") < min(keys)
    assert hidden.any() and torch.equal(out[hidden], clean[hidden])
    if up <= 20 and dtype == BF:
        close(out, (q, k8, v8, ks, far, table, q_start, kv_len), cap)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("up", [20, 100])
def test_large_values_behind_a_window(up, D, dtype):
    m, n, window = 150, 400, 90
    q, k8, v8, ks, vs, table, q_start, kv_len = qc.paged_inputs([m], [n], 8, 2, D, 16, dtype, window=window)
    clean = op(q, k8, v8, ks, vs, table, q_start, kv_len, 0.0, 0.0, window)
    far, key = vs.clone(), n - m - window + 5  # only the first queries see it
    far[table[0, key // 16].long(), key % 16] *= 2.0**up
    out = op(q, k8, v8, ks, far, table, q_start, kv_len, 0.0, 0.0, window)
    hidden = torch.arange(n - m, n, device="cuda") >= key + window
    assert torch.equal(out[hidden], clean[hidden])


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("m", [1, 20, 150])
@pytest.mark.parametrize("up", [16, 30, 60])
def test_large_values_without_weight(up, m, D, dtype):
    """A key of a score 80 nats below the others' and values 2^up times theirs: its share is below
    2^(up - 115) of theirs."""
    n = 300
    q, kc, vc, table, q_start, kv_len = ref.paged_inputs([m], [n], 8, 2, D, 16, dtype)
    q = torch.zeros_like(q)
    q[..., 0] = 8.0
    q[..., 1] = 1.0
    kc[..., 0] = 0.0
    at = table[0, 8].long(), 3
    kc[at[0], at[1], :, 0] = -80.0 * D**0.5 / 8.0
    (k8, ks), (v8, vs) = qc.quantised(kc), qc.quantised(vc)
    vs[at] *= 2.0**up
    x = (q, k8, v8, ks, vs, table, q_start, kv_len)
    close(op(*x), x)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("spread", [0, 6, 10])
@pytest.mark.parametrize("m", [1, 7, 90, 300])
def test_value_scales_apart(m, spread, dtype, D):
    x = qc.paged_inputs([m, 1, 33], [300, 77, 200], 8, 2, D, 16, dtype, spread=spread)
    close(op(*x), x)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("m", [1, 150])
def test_blocks_of_other_sizes(m, dtype):
    """Every page of 16 keys 2^-40 .. 2^8 times the others, the largest ones seen by the last queries alone."""
    n = 256
    q, k8, v8, ks, vs, table, q_start, kv_len = qc.paged_inputs([m], [n], 4, 2, 64, 16, dtype)
    vs = vs.clone()
    for i in range(n // 16):
        vs[table[0, i].long()] *= 2.0 ** (8 - 3 * (n // 16 - 1 - i))
    x = (q, k8, v8, ks, vs, table, q_start, kv_len)
    close(op(*x), x)
