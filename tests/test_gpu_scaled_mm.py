"""b200::scaled_mm (block-scaled e4m3 product) against the formula in 64 bits.

Bound: a product of two e4m3 values is exact in fp32; the tensor core's sum of
128 of them, the products with the scales and the sum over the blocks are
taken as one chain of K + 3 blocks additions that each err by a step of fp32,
2^-23, of the magnitudes' sum; then half a step of the output's type."""
import pytest
import torch

import quant_reference as ref
from serving_reference import HALF_STEP
from compiler import runtime
from compiler.runtime import cabi

pytestmark = pytest.mark.gpu
runtime.load()
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def make(m, k, n, seed=0):
    g = torch.Generator("cuda").manual_seed(seed + m * 7 + k * 3 + n)
    ld = -(-k // 16) * 16
    a, w = ref.random_codes(m, ld, g)[:, :k], ref.random_codes(n, ld, g)[:, :k]
    blocks = -(-k // 128)
    sa = ref.random_scales(m, blocks, g=g)
    sb = ref.random_scales(-(-n // 128), blocks, g=g)
    return a, w.t(), sa, sb.t()


def check(out, a, b, sa, sb):
    want, size = ref.scaled_mm(a, b, sa, sb)
    k = a.shape[1]
    chain = (k + 3 * -(-k // 128)) * 2.0**-23
    tiny = 2.0**-24 if out.dtype == torch.float16 else 0.0
    h = HALF_STEP[out.dtype]
    assert out.shape == want.shape
    assert ((out.double() - want).abs() <= want.abs() * h + size * chain * (1 + h) + tiny).all()


SHAPES = [(1, 128, 64), (1, 8192, 2048), (3, 16, 1), (7, 144, 40), (64, 4096, 256), (128, 512, 130), (129, 1024, 65),
          (200, 640, 300), (257, 384, 513), (777, 2064, 1004), (1000, 100, 1000), (2048, 2048, 2048)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_against_the_formula(m, k, n, dtype):
    a, b, sa, sb = make(m, k, n)
    check(torch.ops.b200.scaled_mm(a, b, sa, sb, dtype), a, b, sa, sb)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,n", [(1, 256, 64), (100, 1152, 200), (300, 2000, 520), (513, 128, 264), (600, 896, 1028)])
@pytest.mark.parametrize("tile,split", [(1, 0), (16, 1), (16, 8), (32, 1), (32, 3), (64, 1), (64, 2), (64, 7), (128, 1), (128, 4)])
def test_every_tile(tile, split, m, k, n, dtype):
    a, b, sa, sb = make(m, k, n)
    out = torch.full((m + 2, n), 7.0, device="cuda", dtype=dtype)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    cabi.scaled_mm(a, b, sa, sb, out[:m], tile=tile, split=split, status=status)
    assert status.item() == 0
    check(out[:m], a, b, sa, sb)
    assert (out[m:] == 7.0).all()  # nothing behind the last row


def test_many_tiles():
    """More tiles than CTAs: the persistent loop, buffers in every phase."""
    a, b, sa, sb = make(3000, 1408, 4000)
    check(torch.ops.b200.scaled_mm(a, b, sa, sb, torch.bfloat16), a, b, sa, sb)
    a, b, sa, sb = make(2500, 128, 5000)
    check(torch.ops.b200.scaled_mm(a, b, sa, sb, torch.float32), a, b, sa, sb)


def test_strided_operands():
    """Columns of wider tensors, scales of any strides; what lies beside is not read."""
    a0, b0, sa0, sb0 = make(70, 1024, 400)
    a0.view(torch.uint8)[:, 512:] = 0x7F  # NaN
    a, b = a0[:, :500], b0[:500]
    sa, sb = sa0[:, :4].t().contiguous().t(), sb0[:4].contiguous()
    check(torch.ops.b200.scaled_mm(a, b, sa, sb, torch.bfloat16), a, b, sa, sb)
    a, sa = a0[::2, :500], sa0[::2, :4]
    check(torch.ops.b200.scaled_mm(a, b, sa, sb, torch.bfloat16), a, b, sa, sb)


@pytest.mark.parametrize("m,tile,split", [(5, 16, 4), (200, 128, 2), (300, 1, 0), (40, 64, 1)])
def test_nan_and_infinity(m, tile, split):
    """A NaN code and a NaN scale reach the rows and columns that they enter, and no others."""
    a, b, sa, sb = make(m, 768, 320)
    a, b, sa, sb = a.clone(), b.t().clone().t(), sa.clone(), sb.clone()
    a.view(torch.uint8)[2, 300] = 0x7F
    b.view(torch.uint8)[5, 100] = 0xFF
    sa[1, 3] = float("nan")
    sb[2, 2] = float("inf")
    out = torch.empty(m, 320, device="cuda", dtype=torch.float32)
    cabi.scaled_mm(a, b, sa, sb, out, tile=tile, split=split)
    bad = torch.zeros(m, 320, dtype=torch.bool, device="cuda")
    bad[1:3] = True
    bad[:, 100] = True
    assert torch.equal(out.isnan()[:, :256], bad[:, :256])
    assert out[~bad[:, 0], 256:].abs().eq(float("inf")).logical_or(out[~bad[:, 0], 256:].isnan()).all()
    assert out[1:3].isnan().all()


def test_empty():
    e = dict(device="cuda", dtype=ref.E4M3)
    s = lambda *shape: torch.ones(*shape, device="cuda")  # noqa: E731
    mm = torch.ops.b200.scaled_mm
    assert mm(torch.empty(0, 256, **e), torch.empty(64, 256, **e).t(), s(0, 2), s(2, 1), torch.bfloat16).shape == (0, 64)
    assert mm(torch.empty(3, 256, **e), torch.empty(0, 256, **e).t(), s(3, 2), s(2, 0), torch.bfloat16).shape == (3, 0)
    out = mm(torch.empty(3, 0, **e), torch.empty(5, 0, **e).t(), s(3, 0), s(0, 1), torch.float32)
    assert out.shape == (3, 5) and (out == 0).all()


def test_same_bits_again_and_in_a_graph():
    a, b, sa, sb = make(48, 4096, 1024)
    want = torch.ops.b200.scaled_mm(a, b, sa, sb, torch.bfloat16)
    assert torch.equal(torch.ops.b200.scaled_mm(a, b, sa, sb, torch.bfloat16), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = torch.ops.b200.scaled_mm(a, b, sa, sb, torch.bfloat16)
    a2, _, sa2, _ = make(48, 4096, 1024, seed=5)
    first = a.clone(), sa.clone()
    a.copy_(a2)
    sa.copy_(sa2)
    graph.replay()
    check(out, a, b, sa, sb)
    a.copy_(first[0])
    sa.copy_(first[1])
    graph.replay()
    assert torch.equal(out, want)


def test_two_streams():
    pairs = [make(200, 1024, 640, seed=s) for s in range(2)]
    streams = [torch.cuda.Stream() for _ in pairs]
    torch.cuda.synchronize()
    outs = []
    for _ in range(5):
        for st, args in zip(streams, pairs):
            with torch.cuda.stream(st):
                outs.append((torch.ops.b200.scaled_mm(*args, torch.bfloat16), args))
    torch.cuda.synchronize()
    for out, args in outs:
        check(out, *args)


@pytest.mark.parametrize("tile,split,m", [(1, 0, 600), (128, 1, 200), (32, 4, 30), (16, 8, 5)])
def test_a_wait_that_runs_out_is_reported(tile, split, m):
    """The first block is never signalled: the kernel reports, drains and
    returns, and the next call is right."""
    a, b, sa, sb = make(m, 1024, 512)
    out = torch.empty(m, 512, device="cuda", dtype=torch.bfloat16)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    cabi.scaled_mm(a, b, sa, sb, out, tile=tile, split=split, status=status, timeout_ns=20_000_000, test_flags=1)
    torch.cuda.synchronize()
    assert status.item() == 6
    status.zero_()
    cabi.scaled_mm(a, b, sa, sb, out, tile=tile, split=split, status=status)
    assert status.item() == 0
    check(out, a, b, sa, sb)
