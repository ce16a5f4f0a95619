"""Replayed graphs and the caches they are given: caches that the caller frees,
replaces or swaps after a graph was recorded with them."""
import gc
import weakref

import pytest
import torch

from compiler import graph_replay, runtime

runtime.load()
STEPS = 4  # decode steps with one set of caches: op by op, recorded, replayed


@pytest.fixture
def records(monkeypatch):
    seen = []
    orig = graph_replay.GraphReplay._record

    def record(self, args):
        seen.append(self)
        orig(self, args)

    monkeypatch.setattr(graph_replay.GraphReplay, "_record", record)
    return seen


class Decode:
    """A compiled stack of four decoder layers next to the eager one, a step of
    single tokens of two sequences at a time."""

    def __init__(self):
        from compiler.backend import custom_backend
        from test_inplace_append import _model

        self.step, self.model = _model(4)
        torch._dynamo.reset()
        self.compiled = torch.compile(self.model, backend=custom_backend, dynamic=False)
        self.cos, self.sin = (torch.randn(64, self.step.D // 2, device="cuda") for _ in range(2))
        self.at = 0

    def caches(self, extra=0):
        """One set (K and V a layer), all with the same pages."""
        sets = [self.step.Cache([40, 40]) for _ in range(4)]
        pad = lambda t: torch.cat([t, t.new_zeros(extra, *t.shape[1:])]) if extra else t  # noqa: E731
        self.index = sets[0]
        return [(pad(c.k), pad(c.v)) for c in sets]

    def run(self, f, caches, x, at):
        pos, slots, _, _, table, q_start, kv_len = self.index.step([(at, at + 1)] * 2)
        with torch.no_grad():
            return f(x, self.cos, self.sin, caches, (pos, slots, table, q_start, kv_len))

    def both(self, mine, eager):
        x = torch.randn(2, self.step.DIM, device="cuda").to(torch.bfloat16)
        got, want = self.run(self.compiled, mine, x, self.at), self.run(self.model, eager, x, self.at)
        self.at += 1
        assert torch.equal(got, want)


def copy(caches):
    return [(k.clone(), v.clone()) for k, v in caches]


@pytest.mark.gpu
def test_replaced_caches_are_released_and_recorded_again(records):
    """The graph keeps no cache alive, and replays again with the new ones."""
    d = Decode()
    mine = d.caches(extra=2000)
    eager = copy(mine)
    for _ in range(STEPS):
        d.both(mine, eager)
    assert len(records) == 1
    for round_ in range(2):
        new = copy(mine)
        old = [weakref.ref(t) for pair in mine for t in pair]
        torch.cuda.synchronize()
        held = torch.cuda.memory_allocated()
        size = sum(t.numel() * 2 for pair in mine for t in pair)
        del mine
        gc.collect()
        assert not any(r() is not None for r in old)
        assert held - torch.cuda.memory_allocated() >= size
        mine = new
        for _ in range(STEPS - 1):
            d.both(mine, eager)
        before = graph_replay.REPLAYS
        d.both(mine, eager)
        assert graph_replay.REPLAYS == before + 1
        assert len(records) == 2 + round_


@pytest.mark.gpu
def test_caches_that_take_turns(records):
    """Two sets in turn: one is replayed, the other runs op by op, and nothing
    is recorded over and over."""
    d = Decode()
    a, b = d.caches(), d.caches()
    eager = copy(a), copy(b)
    for _ in range(8):
        at = d.at
        d.both(a, eager[0])
        d.at = at
        d.both(b, eager[1])
    assert len(records) <= 2
    for mine, want in ((a, eager[0]), (b, eager[1])):
        for s, t in zip(mine, want):
            for x, y in zip(s, t):
                assert torch.equal(x.view(torch.int16), y.view(torch.int16))


@pytest.mark.gpu
def test_caches_replaced_again_and_again_are_recorded_a_bounded_number_of_times(records):
    d = Decode()
    mine = d.caches()
    eager = copy(mine)
    keep = []  # so that no address comes back
    for _ in range(graph_replay.MAX_RECORDS + 3):
        keep.append(mine)
        mine = copy(mine)
        for _ in range(2):
            d.both(mine, eager)
    assert len(records) == graph_replay.MAX_RECORDS


# ------------------------------------------------- caches that a graph only reads
def reader(n=17):
    """Attends `n` times over what `get` makes of its caches."""
    def f(q, caches, table, q_start, kv_len):
        for i in range(n):
            kc, vc = caches[i % len(caches)]
            q = torch.ops.b200.paged_attention(q, kc, vc, table, q_start, kv_len) + q
        return q
    return f


def halves(q, both, table, q_start, kv_len):
    """K and V of a page side by side in one tensor, taken apart in the graph."""
    return reader()(q, [(both[:, 0], both[:, 1])], table, q_start, kv_len)


def traced(f, *args):
    """The graph that AOTAutograd hands to the inference compiler, on fake tensors."""
    from torch._dynamo.backends.common import aot_autograd
    from torch._functorch.aot_autograd import make_boxed_func
    from torch._subclasses.fake_tensor import FakeTensorMode

    seen = []

    def keep(gm, _):
        seen.append(gm)
        return make_boxed_func(gm.forward)

    torch._dynamo.reset()
    with torch.no_grad(), FakeTensorMode(allow_non_fake_inputs=True):
        fake = torch.utils._pytree.tree_map(lambda t: torch.empty(t.shape, dtype=t.dtype, device="cuda"), args)
        torch.compile(f, backend=aot_autograd(fw_compiler=keep, inference_compiler=keep))(*fake)
    torch._dynamo.reset()
    return seen[0]


def cpu_inputs(shape):
    i32 = dict(dtype=torch.int32)
    return (torch.empty(3, 8, 64, dtype=torch.bfloat16), torch.empty(shape, dtype=torch.bfloat16),
            torch.empty(2, 4, **i32), torch.empty(3, **i32), torch.empty(2, **i32))


def attended_shapes(gm):
    from compiler.optimization.inplace_append import attended_inputs

    inputs = [n for n in gm.graph.nodes if n.op == "placeholder"]
    return sorted(tuple(inputs[i].meta["val"].shape) for i in attended_inputs(gm))


def test_inputs_that_are_caches_alone_are_found():
    q, cache, *index = cpu_inputs((9, 16, 2, 64))
    two = lambda q, k, v, *index: reader()(q, [(k, v)], *index)  # noqa: E731
    assert attended_shapes(traced(two, q, cache, cache.clone(), *index)) == [(9, 16, 2, 64)] * 2
    q, both, *index = cpu_inputs((9, 2, 16, 2, 64))
    assert attended_shapes(traced(halves, q, both, *index)) == [(9, 2, 16, 2, 64)]


def test_inputs_that_are_more_than_caches_are_not():
    q, cache, *index = cpu_inputs((9, 16, 2, 64))
    summed = lambda q, k, v, *index: (reader()(q, [(k, v)], *index), k.sum())  # noqa: E731
    assert attended_shapes(traced(summed, q, cache, cache.clone(), *index)) == [(9, 16, 2, 64)]  # v
    seen = lambda q, k, v, *index: (reader()(q, [(k, v)], *index), k[0], v[1:])  # noqa: E731
    assert attended_shapes(traced(seen, q, cache, cache.clone(), *index)) == []
    asked = lambda q, *index: reader()(q, [(q.view(3, 1, 8, 64), q.view(3, 1, 8, 64))], *index)  # noqa: E731
    assert attended_shapes(traced(asked, q, *index)) == []


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["two", "halves"])
def test_replays_read_caches_in_place(layout, records):
    """No copy of a cache is made or kept, changes of its contents are seen, and
    other caches are too."""
    import serving_reference as ref
    from compiler.backend import custom_backend

    q, kc, vc, *index = ref.paged_inputs([1, 2], [40, 30], 8, 2, 64, 16, torch.bfloat16,
                                         layout="pair" if layout == "halves" else "nhd", spare=20000)
    if layout == "halves":
        f, base = halves, kc._base
        make = lambda t: (t,)  # noqa: E731
    else:
        f = lambda q, k, v, *index: reader()(q, [(k, v)], *index)  # noqa: E731
        base = torch.stack([kc, vc])
        make = lambda t: (t[0], t[1])  # noqa: E731
    size = kc.numel() * 2
    torch._dynamo.reset()
    compiled = torch.compile(f, backend=custom_backend, dynamic=False)
    keep = []
    with torch.no_grad():
        for i in range(10):
            if i in (3, 8):
                base[:5] *= 0.5  # the caches' contents
            if i == 5:
                keep.append(base)
                base = base.clone()
            torch.cuda.synchronize()
            torch.cuda.reset_peak_memory_stats()
            start, before = torch.cuda.memory_allocated(), graph_replay.REPLAYS
            got = compiled(q, *make(base), *index)
            torch.cuda.synchronize()
            assert torch.cuda.max_memory_allocated() - start < size
            assert torch.equal(got, f(q, *make(base), *index))
            assert graph_replay.REPLAYS - before == (0 if i in (0, 5) else 1)
    assert len(records) == 2
