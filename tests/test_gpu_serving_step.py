"""The serving operators together, as a decoder layer uses them: residual
addition and norm, projections, rotary append, attention over the pages, for
a prompt in two chunks and single tokens after it, against the same layer in
plain 64-bit PyTorch without a cache; eagerly, as one replayed CUDA graph and
through torch.compile with the backend."""
import math

import pytest
import torch

from compiler import runtime
from compiler.backend import custom_backend

pytestmark = pytest.mark.gpu
runtime.load()
H, HKV, D, DIM, PAGE = 8, 2, 64, 512, 16
BF = torch.bfloat16


class Layer(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.norm1 = torch.nn.Parameter(1 + 0.1 * torch.randn(DIM))
        self.norm2 = torch.nn.Parameter(1 + 0.1 * torch.randn(DIM))
        self.qkv = torch.nn.Linear(DIM, (H + 2 * HKV) * D, bias=False)
        self.o = torch.nn.Linear(H * D, DIM, bias=False)

    def forward(self, x, residual, cos, sin, pos, slots, kc, vc, table, q_start, kv_len):
        ops = torch.ops.b200
        h, residual = ops.add_rms_norm(x, residual, self.norm1, 1e-5)
        q, k, v = (t.unflatten(1, (-1, D)) for t in self.qkv(h).split([H * D, HKV * D, HKV * D], 1))
        q = ops.rope_append(q, k, v, cos, sin, pos, slots, kc, vc)
        a = ops.paged_attention(q, kc, vc, table, q_start, kv_len)
        out, residual = ops.add_rms_norm(self.o(a.flatten(1)), residual, self.norm2, 1e-5)
        return out, residual


def plain(layer, x, residual, cos, sin):
    """The whole sequence at once, 64 bits, [tokens, DIM]."""
    def norm(t, w):
        return t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-5) * w.double()

    r = x.double() + residual.double()
    q, k, v = (norm(r, layer.norm1) @ layer.qkv.weight.double().T).split([H * D, HKV * D, HKV * D], 1)

    def turn(t):
        t = t.unflatten(1, (-1, D))
        a, b = t[..., :D // 2], t[..., D // 2:]
        c, s = cos.double()[:len(t), None], sin.double()[:len(t), None]
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    q, k, v = turn(q), turn(k).repeat_interleave(H // HKV, 1), v.unflatten(1, (-1, D)).repeat_interleave(H // HKV, 1)
    s = torch.einsum("thd,nhd->htn", q, k) / math.sqrt(D)
    s = s.masked_fill(torch.ones(len(x), len(x), dtype=torch.bool, device=x.device).triu(1), -math.inf)
    a = torch.einsum("htn,nhd->thd", s.softmax(-1), v).flatten(1)
    r = r + a @ layer.o.weight.double().T
    return norm(r, layer.norm2), r


class Cache:
    """Two sequences whose pages interleave, in a cache full of NaN."""

    def __init__(self, lengths):
        pages = sum(-(-n // PAGE) for n in lengths) + 1
        self.k, self.v = (torch.full((pages, PAGE, HKV, D), float("nan"), device="cuda", dtype=BF) for _ in range(2))
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(3)).tolist()
        self.table = torch.full((len(lengths), max(-(-n // PAGE) for n in lengths)), -1, dtype=torch.int32)
        for b, n in enumerate(lengths):
            for i in range(-(-n // PAGE)):
                self.table[b, i] = order.pop()
        self.host = self.table.clone()
        self.table = self.table.cuda()

    def step(self, spans):
        """Index tensors for the tokens [lo, hi) of each sequence."""
        pos = [p for lo, hi in spans for p in range(lo, hi)]
        slots = [int(self.host[b, p // PAGE]) * PAGE + p % PAGE for b, (lo, hi) in enumerate(spans) for p in range(lo, hi)]
        starts = [0]
        for lo, hi in spans:
            starts.append(starts[-1] + hi - lo)
        i32 = dict(dtype=torch.int32, device="cuda")
        return (torch.tensor(pos, **i32), torch.tensor(slots, device="cuda"), self.k, self.v, self.table,
                torch.tensor(starts, **i32), torch.tensor([hi for _, hi in spans], **i32))


@pytest.fixture(scope="module")
def setting():
    torch.manual_seed(0)
    layer = Layer().to("cuda", BF).requires_grad_(False)
    lengths = [203, 150]
    x, res = (torch.randn(sum(lengths), DIM, device="cuda").to(BF) for _ in range(2))
    angle = torch.outer(torch.arange(256, device="cuda").double(), 10000.0 ** (-torch.arange(0, D, 2, device="cuda") / D))
    cos, sin = angle.cos().float(), angle.sin().float()
    want = [plain(layer, a, b, cos, sin) for a, b in zip(x.split(lengths), res.split(lengths))]
    return layer, lengths, x.split(lengths), res.split(lengths), cos, sin, want


def spans_of(lengths):
    """Two prompt chunks (the second sequence ends earlier), then single tokens."""
    yield [(0, 96), (0, 70)]
    yield [(96, 200), (70, 147)]
    for i in range(3):
        yield [(200 + i, 201 + i), (147 + i, 148 + i)]


def run(setting, call):
    layer, lengths, x, res, cos, sin, want = setting
    cache = Cache(lengths)
    got = [[], []]
    for spans in spans_of(lengths):
        xs = torch.cat([x[b][lo:hi] for b, (lo, hi) in enumerate(spans)])
        rs = torch.cat([res[b][lo:hi] for b, (lo, hi) in enumerate(spans)])
        out, r = call(layer, xs, rs, cos, sin, *cache.step(spans))
        at = 0
        for b, (lo, hi) in enumerate(spans):
            got[b].append((out[at:at + hi - lo].clone(), r[at:at + hi - lo].clone()))
            at += hi - lo
    for b in range(2):
        for i in range(2):
            mine, ref = torch.cat([g[i] for g in got[b]]).double(), want[b][i]
            # bf16 between the steps: six roundings (sum, norm, projection,
            # q/k/v, attention, projection) of half a step, 2^-8 of the values,
            # in the norm of all of them: below 8 * 2^-8 / sqrt(3) relative
            assert ((mine - ref).norm() / ref.norm()).item() < 8 * 2.0**-8 / 3**0.5
    assert runtime.gemm_status() == 0


def test_eager(setting):
    run(setting, lambda layer, *a: layer(*a))


def test_compiled(setting):
    torch._dynamo.reset()
    compiled = torch.compile(setting[0], backend=custom_backend, dynamic=False)
    with torch.no_grad():
        run(setting, lambda layer, *a: compiled(*a))


def test_replayed_decode_steps(setting):
    """A captured single-token step, replayed for each token with the step's
    inputs and index tensors copied in."""
    state = {}

    def call(layer, *a):
        if a[0].shape[0] != 2:
            return layer(*a)
        if not state:
            state["in"] = [t.clone() if t.data_ptr() not in (a[6].data_ptr(), a[7].data_ptr()) else t for t in a]
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                layer(*state["in"])
            torch.cuda.current_stream().wait_stream(side)
            state["graph"] = torch.cuda.CUDAGraph()
            with torch.cuda.graph(state["graph"]):
                state["out"] = layer(*state["in"])
        for dst, src in zip(state["in"], a):
            if dst.data_ptr() != src.data_ptr():
                dst.copy_(src)
        state["graph"].replay()
        return state["out"]

    run(setting, call)


@pytest.mark.parametrize("backend", ["aot_eager", custom_backend])
def test_a_training_graph_is_refused(backend):
    x, r = (torch.randn(4, DIM, device="cuda").to(BF) for _ in range(2))
    w = torch.ones(DIM, device="cuda", requires_grad=True)

    def f(x, r, w):
        return torch.ops.b200.add_rms_norm(x * 2, r, w, 1e-5)[0] + x

    torch._dynamo.reset()
    g = torch.compile(f, backend=backend)
    with pytest.raises(Exception, match="no gradient is defined"):
        g(x, r, w)
    with torch.no_grad():
        assert torch.equal(g(x, r, w), f(x, r, w))
