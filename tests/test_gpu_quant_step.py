"""The 8-bit operators together, as a decoder layer uses them: norm with an e4m3
output, block-scaled products, rotary append to an e4m3 cache, attention over it,
SwiGLU with an e4m3 output; for a prompt in two chunks and single tokens after
it.  Each stage is held to its formula in 64 bits on what the stage before
really left; the whole is the same bits eagerly, as a replayed CUDA graph and
through torch.compile with the backend."""
import pytest
import torch

import quant_cache as qc
import quant_reference as quant
import serving_reference as ref
from compiler import graph_replay, runtime
from compiler.backend import custom_backend
from test_gpu_serving_step import spans_of

pytestmark = pytest.mark.gpu
runtime.load()
H, HKV, D, DIM, FFN, PAGE = 8, 2, 64, 512, 896, 16
BF = torch.bfloat16


class Linear8(torch.nn.Module):
    """A linear layer's weight [n, k] in e4m3, a scale for each 128 x 128 block."""

    def __init__(self, k, n):
        super().__init__()
        w = torch.randn(n, k) * k**-0.5
        scale = torch.stack([torch.stack([b.abs().amax() for b in r.split(128, 1)]) for r in w.split(128)]) / quant.MAX
        wide = quant.spread(quant.spread(scale, k).t(), n).t()
        self.register_buffer("weight", (w / wide).clamp(-quant.MAX, quant.MAX).to(quant.E4M3))
        self.register_buffer("scale", scale)

    def forward(self, x8, xs):
        return torch.ops.b200.scaled_mm(x8, self.weight.t(), xs, self.scale.t(), BF)


class Layer(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.norm1 = torch.nn.Parameter((1 + 0.1 * torch.randn(DIM)).to(BF))
        self.norm2 = torch.nn.Parameter((1 + 0.1 * torch.randn(DIM)).to(BF))
        self.qkv, self.o = Linear8(DIM, (H + 2 * HKV) * D), Linear8(H * D, DIM)
        self.gate_up, self.down = Linear8(DIM, 2 * FFN), Linear8(FFN, DIM)

    def forward(self, x, residual, cos, sin, pos, slots, caches, table, q_start, kv_len, seen=None):
        ops = torch.ops.b200
        h, hs, residual = ops.add_rms_norm_quant(x, residual, self.norm1, 1e-5, 128)
        qkv = self.qkv(h, hs)
        q, k, v = (t.unflatten(1, (-1, D)) for t in qkv.split([H * D, HKV * D, HKV * D], 1))
        q = ops.rope_append_quant(q, k, v, cos, sin, pos, slots, *caches)
        a = ops.paged_attention_quant(q, *caches, table, q_start, kv_len)
        a8, as_ = ops.quant_groups(a.flatten(1))
        o = self.o(a8, as_)
        h2, hs2, residual = ops.add_rms_norm_quant(o, residual, self.norm2, 1e-5, 128)
        gu = self.gate_up(h2, hs2)
        f8, fs = ops.quant_groups(gu, True)
        out = self.down(f8, fs)
        if seen is not None:
            seen.update(h=h, hs=hs, qkv=qkv, q=q, a=a, a8=a8, as_=as_, o=o, h2=h2, hs2=hs2, gu=gu, f8=f8, fs=fs, out=out)
        return out, residual


class Cache:
    """Two sequences whose pages interleave, in a cache full of NaN."""

    def __init__(self, lengths):
        pages = sum(-(-n // PAGE) for n in lengths) + 1
        codes = [torch.full((pages, PAGE, HKV, D), 0x7F, device="cuda", dtype=torch.uint8).view(quant.E4M3) for _ in range(2)]
        scales = [torch.full((pages, HKV, PAGE), float("nan"), device="cuda").transpose(1, 2) for _ in range(2)]
        self.all = (*codes, *scales)
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(3)).tolist()
        self.host = torch.full((len(lengths), max(-(-n // PAGE) for n in lengths)), -1, dtype=torch.int32)
        for b, n in enumerate(lengths):
            for i in range(-(-n // PAGE)):
                self.host[b, i] = order.pop()
        self.table = self.host.cuda()

    def step(self, spans):
        pos = [p for lo, hi in spans for p in range(lo, hi)]
        slots = [int(self.host[b, p // PAGE]) * PAGE + p % PAGE for b, (lo, hi) in enumerate(spans) for p in range(lo, hi)]
        starts = [0]
        for lo, hi in spans:
            starts.append(starts[-1] + hi - lo)
        i32 = dict(dtype=torch.int32, device="cuda")
        return (torch.tensor(pos, **i32), torch.tensor(slots, device="cuda"), self.all, self.table, torch.tensor(starts, **i32),
                torch.tensor([hi for _, hi in spans], **i32))


@pytest.fixture(scope="module")
def setting():
    torch.manual_seed(0)
    layer = Layer().to("cuda").requires_grad_(False)
    lengths = [203, 150]
    x, res = (torch.randn(sum(lengths), DIM, device="cuda").to(BF).split(lengths) for _ in range(2))
    angle = torch.outer(torch.arange(256, device="cuda").double(), 10000.0 ** (-torch.arange(0, D, 2, device="cuda") / D))
    return layer, lengths, x, res, angle.cos().float(), angle.sin().float()


def steps(setting):
    layer, lengths, x, res, cos, sin = setting
    cache = Cache(lengths)
    for spans in spans_of(lengths):
        part = [torch.cat([t[lo:hi] for t, (lo, hi) in zip(xs, spans)]) for xs in (x, res)]
        yield (*part, cos, sin, *cache.step(spans))


def mm_close(got, linear, x8, xs):
    want, size = quant.scaled_mm(x8, linear.weight.t(), xs, linear.scale.t())
    k = x8.shape[1]
    chain = (k + 3 * -(-k // 128)) * 2.0**-23
    assert ((got.double() - want).abs() <= want.abs() * 2.0**-8 + size * chain * 1.01).all()


def quant_close(codes, scale, y, err):
    z = y / quant.spread(scale.double(), y.shape[-1])
    assert ((codes.double() - z).abs() <= quant.code_step(z) + z.abs() * err).all()


def test_every_stage_against_its_formula(setting):
    layer = setting[0]
    for args in steps(setting):
        x, res, cos, sin, pos, slots, caches, table, q_start, kv_len = args
        s = {}
        out, residual = layer(*args, seen=s)
        total, y = ref.add_rms_norm(x, res, layer.norm1, 1e-5)
        quant_close(s["h"], s["hs"], y, 3e-5)
        mm_close(s["qkv"], layer.qkv, s["h"], s["hs"])
        q, k, v = (t.unflatten(1, (-1, D)) for t in s["qkv"].split([H * D, HKV * D, HKV * D], 1))
        at = slots // PAGE, slots % PAGE
        kept = [c.view(torch.uint8)[at].view(quant.E4M3) if c.dtype == quant.E4M3 else c[at] for c in caches]
        for codes, scale, row in ((kept[0], kept[2], ref.rotate(k, cos[pos.long()], sin[pos.long()])[0]), (kept[1], kept[3], v.double())):
            z = row / scale.double()[..., None]
            assert ((codes.double() - z).abs() <= quant.code_step(z) + 448 * 2.0**-20).all()
        qc.attention_close(s["a"], (s["q"], *caches, table, q_start, kv_len), ref.default_scale(D))
        quant_close(s["a8"], s["as_"], s["a"].flatten(1).double(), 2.0**-21)
        mm_close(s["o"], layer.o, s["a8"], s["as_"])
        total, y = ref.add_rms_norm(s["o"], total, layer.norm2, 1e-5)
        assert torch.equal(residual, total)
        quant_close(s["h2"], s["hs2"], y, 3e-5)
        mm_close(s["gu"], layer.gate_up, s["h2"], s["hs2"])
        quant_close(s["f8"], s["fs"], quant.silu_mul(s["gu"]), 1e-5)
        mm_close(out, layer.down, s["f8"], s["fs"])
    runtime.check_status()


def test_captured_and_replayed(setting):
    layer = setting[0]
    eager = [layer(*args) for args in steps(setting)]
    got = []
    for args in steps(setting):
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            out = layer(*args)
        g.replay()
        got.append([t.clone() for t in out])
    for a, b in zip(eager, got):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("layers", [1, 3])  # below and above the launches that a graph is replayed from
def test_compiled_steps_equal_eager_ones(setting, layers):
    class Stack(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.layers = torch.nn.ModuleList(Layer() for _ in range(layers))

        def forward(self, x, residual, cos, sin, pos, slots, caches, table, q_start, kv_len):
            for layer, c in zip(self.layers, caches):
                x, residual = layer(x, residual, cos, sin, pos, slots, c, table, q_start, kv_len)
            return x, residual

    torch.manual_seed(1)
    _, lengths, x, res, cos, sin = setting
    model = Stack().to("cuda").requires_grad_(False)
    torch._dynamo.reset()
    compiled = torch.compile(model, backend=custom_backend, dynamic=False)
    stores = [[Cache(lengths) for _ in range(layers)] for _ in range(2)]
    before = graph_replay.REPLAYS
    spans = list(spans_of(lengths))
    spans += [[(i, i + 1), (i, i + 1)] for i in range(4)]  # single tokens once more, over the old ones
    with torch.no_grad():
        for sp in spans:
            part = [torch.cat([t[lo:hi] for t, (lo, hi) in zip(xs, sp)]) for xs in (x, res)]
            outs = []
            for f, per in ((compiled, stores[0]), (model, stores[1])):
                idx = [c.step(sp) for c in per]
                pos, slots, _, _, q_start, kv_len = idx[0]
                outs.append(f(*part, cos, sin, pos, slots, [c.all for c in per], per[0].table, q_start, kv_len))
            assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
    for a, b in zip(*stores):
        for s, t in zip(a.all, b.all):
            raw = torch.uint8 if s.dtype == quant.E4M3 else torch.int32
            assert torch.equal(s.contiguous().view(raw), t.contiguous().view(raw))
    assert (graph_replay.REPLAYS > before) == (layers == 3)
    runtime.check_status()
