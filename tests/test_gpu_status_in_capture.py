"""A process whose first library calls are being captured: the captured kernels
report to the status word all the same."""
import os
import subprocess
import sys

import pytest

from compiler.runtime import cabi

pytestmark = pytest.mark.gpu

BODY = """
import sys; sys.path[:0] = [%r, %r]
import torch, serving_reference as ref
from compiler import runtime
runtime.load()
ops = torch.ops.b200
q, kc, vc, table, q_start, kv_len = ref.paged_inputs([1, 300], [90, 300], 8, 2, 64, 16, torch.bfloat16)
slots = torch.zeros(301, dtype=torch.int64, device="cuda")
pos = torch.zeros(301, dtype=torch.int64, device="cuda")
cos = torch.ones(4, 32, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    if %r == "attend":
        out = ops.paged_attention(q, kc, vc, table, q_start, kv_len)
    else:
        out = ops.rope_append(q, q[:, :2], q[:, :2], cos, cos, pos, slots, kc, vc)
g.replay()
assert runtime.gemm_status() == 0
good = table[1, 2].item()
table[1, 2] = 10**6
slots[7] = 10**6
for _ in range(2):  # and again after the word was cleared
    g.replay()
    assert runtime.gemm_status() == 9
g.replay()  # what one replay reports, the next does not clear
table[1, 2] = good
slots[7] = 0
g.replay()
assert runtime.gemm_status() == 9
g.replay()
assert runtime.gemm_status() == 0
print("fine")
"""


@pytest.mark.parametrize("op", ["attend", "append"])
def test_captured_first_calls_report(op):
    here = os.path.dirname(os.path.abspath(__file__))
    package = os.path.dirname(os.path.dirname(os.path.dirname(cabi.__file__)))
    r = subprocess.run([sys.executable, "-c", BODY % (here, package, op)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-2000:]
