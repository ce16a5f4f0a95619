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
