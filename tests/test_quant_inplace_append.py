"""The pass that puts cache appends back in place, for appends to e4m3 caches,
which write their scales too (CPU)."""
import operator

import pytest
import torch
import torch.fx as fx

from compiler import runtime
from compiler.optimization.inplace_append import appended_inputs, attended_inputs, inplace_append

runtime.load()
APPEND = torch.ops.b200.rope_append_quant.default
ATTEND = torch.ops.b200.paged_attention_quant.default
FUNCTIONAL = torch.ops.higher_order.auto_functionalized_v2
NAMES = ("q", "k", "v", "cos", "sin", "positions", "slots")
CACHES = ("k_cache", "v_cache", "k_scale", "v_scale")


def graph(steps, alias=None, order=(0, 1, 2, 3)):
    """Placeholders NAMES, CACHES, table; `alias`: a cache that is a view of its
    input; `order`: where each cache stands among the append's bases."""
    g = fx.Graph()
    p = {n: g.placeholder(n) for n in (*NAMES, *CACHES, "table")}
    state = {c: p[c] for c in CACHES}
    if alias:
        state[alias] = g.call_function(torch.ops.aten.alias.default, (p[alias],))
    outs = []
    for s in steps:
        if s == "append":
            bases = [None] * 4
            for c, i in zip(CACHES, order):
                bases[i] = state[c]
            kw = {**{n: p[n] for n in NAMES}, **{f"_{c}_base_index": i for c, i in zip(CACHES, order)}, "_all_bases": bases}
            a = g.call_function(FUNCTIONAL, (APPEND,), kw)
            outs.append(g.call_function(operator.getitem, (a, 0)))
            state = {c: g.call_function(operator.getitem, (a, 1 + i)) for c, i in zip(CACHES, order)}
        else:
            src = p if s == "attend first state" else state
            outs.append(g.call_function(ATTEND, (p["q"], *(src[c] for c in CACHES), p["table"], p["table"], p["table"])))
    g.output((*(state[c] for c in CACHES), *outs))
    return fx.GraphModule(torch.nn.Module(), g)


def targets(gm):
    return [n.target for n in gm.graph.nodes if n.op == "call_function"]


@pytest.mark.parametrize("order", [(0, 1, 2, 3), (2, 0, 3, 1)])
def test_an_append_and_its_reader_become_in_place(order):
    gm = inplace_append(graph(["append", "attend"], order=order))
    assert targets(gm) == [APPEND, ATTEND]
    nodes = {n.name: n for n in gm.graph.nodes}
    append = next(n for n in gm.graph.nodes if n.target == APPEND)
    assert append.args == tuple(nodes[n] for n in (*NAMES, *CACHES))
    out = next(n for n in gm.graph.nodes if n.op == "output").args[0]
    assert out[:4] == tuple(nodes[c] for c in CACHES)  # the inputs themselves are returned
    assert appended_inputs(gm) == (7, 8, 9, 10)


def test_a_reader_between_appends_is_not_run_twice():
    gm = inplace_append(graph(["append", "attend", "append", "attend"]))
    assert targets(gm) == [APPEND, ATTEND, APPEND, ATTEND] and appended_inputs(gm) is None


@pytest.mark.parametrize("steps,alias", [(["append", "attend first state"], None), (["append"], "k_scale"), (["append"], "v_cache")])
def test_left_functional(steps, alias):
    with pytest.warns(UserWarning, match="b200::rope_append_quant"):
        gm = inplace_append(graph(steps, alias))
    assert FUNCTIONAL in targets(gm) and APPEND not in targets(gm)


def test_caches_that_are_only_attended_over():
    gm = graph(["attend"])
    out = next(n for n in gm.graph.nodes if n.op == "output")
    out.args = (out.args[0][4:],)
    gm.recompile()
    assert inplace_append(gm) is gm and appended_inputs(gm) == () and attended_inputs(gm) == (7, 8, 9, 10)
