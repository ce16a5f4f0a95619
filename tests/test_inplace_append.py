"""Cache appends of compiled graphs in place: the pass's decisions on CPU, and
compiled decode steps (op by op and replayed) on the GPU."""
import operator

import pytest
import torch
import torch.fx as fx

from compiler import graph_replay, runtime
from compiler.optimization import config
from compiler.optimization.inplace_append import appended_inputs, inplace_append

runtime.load()
APPEND = torch.ops.b200.rope_append.default
ATTEND = torch.ops.b200.paged_attention.default
FUNCTIONAL = torch.ops.higher_order.auto_functionalized_v2
NAMES = ("q", "k", "v", "cos", "sin", "positions", "slots")


def graph(steps, returns=("kc", "vc")):
    """Graph over placeholders q k v cos sin positions slots kc vc; `steps`
    names what happens to the caches in order."""
    g = fx.Graph()
    p = {n: g.placeholder(n) for n in (*NAMES, "kc", "vc", "table")}
    state = {"kc": p["kc"], "vc": p["vc"]}
    first = dict(state)
    outs = []
    for s in steps:
        if s == "append":
            a = g.call_function(FUNCTIONAL, (APPEND,), {**{n: p[n] for n in NAMES}, "_k_cache_base_index": 0,
                                                        "_v_cache_base_index": 1, "_all_bases": [state["kc"], state["vc"]]})
            outs.append(g.call_function(operator.getitem, (a, 0)))
            state = {"kc": g.call_function(operator.getitem, (a, 1)), "vc": g.call_function(operator.getitem, (a, 2))}
        elif s == "attend":
            outs.append(g.call_function(ATTEND, (p["q"], state["kc"], state["vc"], p["table"], p["table"], p["table"])))
        elif s == "attend first state":
            outs.append(g.call_function(ATTEND, (p["q"], first["kc"], first["vc"], p["table"], p["table"], p["table"])))
        elif s == "view":
            outs.append(g.call_function(torch.ops.aten.view.default, (state["kc"], [-1])))
        elif s == "view argument":
            state["kc"] = g.call_function(torch.ops.aten.alias.default, (state["kc"],))
    named = {**{n: state[n] for n in state}, "first": first["kc"]}
    g.output((*(named[r] for r in returns), *outs))
    return fx.GraphModule(torch.nn.Module(), g)


def targets(gm):
    return [n.target for n in gm.graph.nodes if n.op == "call_function"]


def test_an_append_and_its_reader_become_in_place():
    gm = inplace_append(graph(["append", "attend"]))
    assert targets(gm) == [APPEND, ATTEND]
    nodes = {n.name: n for n in gm.graph.nodes}
    out = next(n for n in gm.graph.nodes if n.op == "output").args[0]
    assert out[:2] == (nodes["kc"], nodes["vc"])  # the inputs themselves are returned
    assert appended_inputs(gm) == (7, 8)


def test_two_appends_in_a_row():
    gm = inplace_append(graph(["append", "attend", "append", "attend"]))
    assert targets(gm) == [APPEND, ATTEND, APPEND, ATTEND]
    # the reader between them must not see the second append: not to be run twice
    assert appended_inputs(gm) is None


def test_a_reader_before_the_append_is_kept_but_not_run_twice():
    gm = inplace_append(graph(["attend", "append"]))
    assert targets(gm) == [ATTEND, APPEND]
    assert appended_inputs(gm) is None


@pytest.mark.parametrize("steps,returns", [
    (["append", "attend first state"], ("kc", "vc")),  # reads the old state after the append
    (["view", "append"], ("kc", "vc")),                # a view of the old state lives on
    (["view argument", "append"], ("kc", "vc")),       # not a whole input
    (["append"], ("kc", "vc", "first")),               # the old state is returned
])
def test_left_functional(steps, returns):
    gm = inplace_append(graph(steps, returns))
    assert FUNCTIONAL in targets(gm) and APPEND not in targets(gm)


def test_graphs_without_appends_are_not_touched():
    gm = graph(["attend"])
    assert inplace_append(gm) is gm and appended_inputs(gm) == ()


def test_written_inputs_do_not_count_as_outputs():
    gm = inplace_append(graph(["append", "attend"]))
    for n in gm.graph.nodes:
        if n.name in ("kc", "vc"):
            n.meta["val"] = torch.empty(config.GRAPH_MAX_OUTPUT_MB * 2**20, dtype=torch.int8, device="meta")
    assert graph_replay.output_bytes(gm) == 2 * config.GRAPH_MAX_OUTPUT_MB * 2**20
    assert graph_replay.output_bytes(gm, (7, 8)) == 0


def _model(layers):
    import test_gpu_serving_step as step

    class Stack(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.layers = torch.nn.ModuleList(step.Layer() for _ in range(layers))

        def forward(self, x, cos, sin, caches, index):
            r = torch.zeros_like(x)
            pos, slots, table, q_start, kv_len = index
            for layer, (kc, vc) in zip(self.layers, caches):
                x, r = layer(x, r, cos, sin, pos, slots, kc, vc, table, q_start, kv_len)
            return x

    torch.manual_seed(1)
    return step, Stack().to("cuda", torch.bfloat16).requires_grad_(False)


@pytest.mark.gpu
@pytest.mark.parametrize("layers", [1, 4])  # below and above the launches that a graph is replayed from
def test_compiled_steps_append_in_place_and_equal_eager(layers):
    from compiler.backend import custom_backend

    step, model = _model(layers)
    torch._dynamo.reset()
    compiled = torch.compile(model, backend=custom_backend, dynamic=False)
    cos, sin = torch.randn(64, step.D // 2, device="cuda"), torch.randn(64, step.D // 2, device="cuda")
    stores = [[step.Cache([40, 30]) for _ in range(layers)] for _ in range(2)]  # compiled, eager
    big = 64 * 2**20  # what a copy of one enlarged cache would cost at least
    for per in stores:
        for c in per:
            c.k, c.v = (torch.cat([t, t.new_zeros(big // (step.PAGE * step.HKV * step.D * 2), *t.shape[1:])]) for t in (c.k, c.v))
    before = graph_replay.REPLAYS
    with torch.no_grad():
        for i in range(6):
            spans = [(0, 20), (0, 11)] if i == 0 else [(19 + i, 20 + i), (10 + i, 11 + i)]
            x = torch.randn(sum(b - a for a, b in spans), step.DIM, device="cuda").to(torch.bfloat16)
            out = []
            for f, per in ((compiled, stores[0]), (model, stores[1])):
                idx = [c.step(spans) for c in per]
                pos, slots, _, _, table, q_start, kv_len = idx[0]
                for c in per[1:]:
                    c.table = per[0].table
                torch.cuda.synchronize()
                torch.cuda.reset_peak_memory_stats()
                base = torch.cuda.memory_allocated()
                out.append(f(x, cos, sin, [(c.k, c.v) for c in per], (pos, slots, table, q_start, kv_len)))
                torch.cuda.synchronize()
                assert torch.cuda.max_memory_allocated() - base < big
            assert torch.equal(*out)
    for a, b in zip(*stores):
        for s, t in ((a.k, b.k), (a.v, b.v)):
            assert torch.equal(s.view(torch.int16), t.view(torch.int16))
    assert (graph_replay.REPLAYS > before) == (layers == 4)
