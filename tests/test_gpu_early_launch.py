"""The 8-bit operators start under the end of the kernel before them: every input
that this one writes, values, scales, index tensors and tables, is read as it left
them.  Inputs change from call to call in the same memory, nothing waits on the host
in between, and the bits are those of calls that stand alone."""
import pytest
import torch

import quant_cache as qc
import quant_reference as quant
from compiler import runtime
from test_gpu_scaled_mm import make

pytestmark = pytest.mark.gpu
runtime.load()
ops = torch.ops.b200
BF = torch.bfloat16


def raw(t):
    return t.view(torch.uint8) if t.dtype == quant.E4M3 else t


def bits(t):
    return t.contiguous().view(torch.uint8)  # NaN too


def like(t):
    """Memory with t's sizes and strides (t's own elements in between)."""
    return torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=t.device)


def copy(dst, src):
    for d, s in zip(dst, src):
        raw(d).copy_(raw(s))


def mm_case(m):
    def inputs(seed):
        a, b, sa, sb = make(m, 1024, 640, seed=seed)
        return [a, b.t(), sa, sb.t()]

    return inputs, lambda a, w, sa, sb: [ops.scaled_mm(a, w.t(), sa, sb.t(), BF)]


def quant_case(rows, cols, swiglu, dtype=BF):
    def inputs(seed):
        g = torch.Generator("cuda").manual_seed(seed)
        return [torch.randn(rows, cols, device="cuda", generator=g).to(dtype)]

    return inputs, lambda x: list(ops.quant_groups(x, swiglu))


def append_case(tokens, dim, table_type):
    def inputs(seed):
        g = torch.Generator("cuda").manual_seed(seed)
        qkv = [torch.randn(tokens, h, dim, device="cuda", generator=g).to(BF) for h in (8, 2, 2)]
        tables = [torch.randn(64, dim // 4, device="cuda", generator=g).to(table_type) for _ in range(2)]
        pos = torch.randint(0, 64, (tokens,), device="cuda", generator=g)
        slots = torch.randperm(tokens + 30, device="cuda", generator=g)[:tokens].int()
        pages = -(-(tokens + 30) // 16)
        caches = [torch.zeros(pages, 16, 2, dim, device="cuda", dtype=torch.uint8).view(quant.E4M3) for _ in range(2)]
        return [*qkv, *tables, pos, slots, *caches, *(torch.zeros(pages, 16, 2, device="cuda") for _ in range(2))]

    def call(*x):
        return [ops.rope_append_quant(*x), *(t.clone() for t in x[7:])]

    return inputs, call


def attention_case(m, max_q):
    def inputs(seed):
        # the same sizes, lengths handed out another way round by every seed
        ns = [300, 77, 1200, 16, 500]
        q, *caches, table, start, _ = qc.paged_inputs([m] * 5, [1200] * 5, 8, 2, 64, 16, BF, seed=seed)
        return [q, *caches, table, start, torch.tensor(ns[seed % 5:] + ns[:seed % 5], dtype=torch.int32, device="cuda")]

    return inputs, lambda *x: [ops.paged_attention_quant(*x, 0.0, 0.0, 0, max_q)]


CASES = {"mm few rows": mm_case(5), "mm rows": mm_case(100), "mm wide": mm_case(3000), "quant": quant_case(64, 4096, False),
         "quant any": quant_case(64, 4099, False), "quant f32": quant_case(64, 512, False, torch.float32),
         "swiglu": quant_case(700, 2048, True), "append": append_case(40, 64, torch.float32),
         "append many": append_case(5000, 128, BF), "append any": append_case(300, 80, torch.float32),
         "attention": attention_case(1, 1), "attention rows": attention_case(3, 3), "attention tiles": attention_case(60, 0)}


@pytest.mark.parametrize("name", CASES)
def test_inputs_written_by_the_kernel_before(name):
    inputs, call = CASES[name]
    sets = [inputs(s) for s in range(5)]
    want = []
    for x in sets:
        torch.cuda.synchronize()
        want.append(call(*[like(t).copy_(t) if t.dtype != quant.E4M3 else t.clone(memory_format=torch.preserve_format) for t in x]))
        torch.cuda.synchronize()
    static = [like(t) for t in sets[0]]
    far = torch.empty(1 << 26, device="cuda")
    got = []
    for i in range(25):
        if i % 3 == 0:
            far.zero_()  # the queue stays ahead of the GPU
        copy(static, sets[i % 5])
        got.append(call(*static))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        for a, b in zip(g, want[i % 5]):
            assert torch.equal(bits(a), bits(b))


@pytest.mark.parametrize("name", CASES)
def test_inputs_from_two_branches_of_a_graph(name):
    """Captured behind a join: half of the inputs are written on another stream."""
    inputs, call = CASES[name]
    sets = [inputs(s) for s in range(3)]
    want = []
    for x in sets:
        want.append(call(*[t.clone(memory_format=torch.preserve_format) for t in x]))
        torch.cuda.synchronize()
    source = [like(t) for t in sets[0]]
    static = [like(t) for t in sets[0]]
    far = torch.empty(1 << 24, device="cuda")
    copy(source, sets[0])
    copy(static, sets[0])
    call(*static)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            far.zero_()
            copy(static[::2], source[::2])
        copy(static[1::2], source[1::2])
        main.wait_stream(side)
        out = call(*static)
    for i in (1, 2, 0, 1):
        copy(source, sets[i])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want[i]):
            assert torch.equal(bits(a), bits(b))


@pytest.mark.parametrize("down", [1, 32])  # values that overflow on the way, and values that do not
def test_a_chain_of_early_launches(down):
    """Each operator on what the one before left, all launched at once, against the same calls one at a time."""
    g = torch.Generator("cuda").manual_seed(1)
    T, H, KV, D, DIM = 40, 8, 2, 64, 512
    a0, w1, s0, sw1 = make(T, DIM, (H + 2 * KV) * D)
    _, w2, _, sw2 = make(T, H * D, 2 * DIM)
    sw1, sw2 = sw1 / down, sw2 / down
    pages = 12
    caches = [torch.zeros(pages, 16, KV, D, device="cuda", dtype=torch.uint8).view(quant.E4M3) for _ in range(2)]
    scales = [torch.zeros(pages, 16, KV, device="cuda") for _ in range(2)]
    angle = torch.rand(64, D // 2, device="cuda", generator=g)
    pos = torch.arange(T, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    table, start = torch.arange(pages, **i32).view(4, 3), torch.tensor([0, 40, 40, 40, 40], **i32)
    lens = torch.tensor([40, 0, 0, 0], **i32)

    def chain(pause):
        a, s, seen = a0, s0, []
        for _ in range(6):
            qkv = ops.scaled_mm(a, w1, s, sw1, BF)
            pause()
            q, k, v = (t.unflatten(1, (-1, D)) for t in qkv.split([H * D, KV * D, KV * D], 1))
            q = ops.rope_append_quant(q, k, v, angle.cos(), angle.sin(), pos, pos, *caches, *scales)
            pause()
            o = ops.paged_attention_quant(q, *caches, *scales, table, start, lens)
            pause()
            o8, os = ops.quant_groups(o.flatten(1))
            pause()
            y = ops.scaled_mm(o8, w2, os, sw2, BF)
            pause()
            a, s = ops.quant_groups(y, True)
            pause()
            seen += [qkv, q, o, o8, os, y, a, s, *(c.clone() for c in (*caches, *scales))]
        torch.cuda.synchronize()
        return seen

    want = chain(torch.cuda.synchronize)
    for _ in range(5):
        for got, w in zip(chain(lambda: None), want):
            assert torch.equal(bits(got), bits(w))
