"""Cache appends kept in place (an extension: the reference has no op that
writes its inputs).

AOTAutograd makes a graph functional, so ``b200::rope_append``, which writes
its two caches, arrives as ``auto_functionalized_v2``: run as it stands, that
node copies both caches, appends to the copies, and the copies are written
back over the inputs at the end of the call -- three passes over a cache that
may fill most of the GPU's memory, for a few appended rows.  This pass puts
the op itself back wherever that cannot be told apart: the caches are whole
graph inputs (or what an earlier append of the graph left of them), and
nothing that reads the state before the append runs after it.  An append that
stays functional (caches that are parts of a larger tensor: K and V as its
halves, layers stacked) gives the same results; it is warned of, since the
whole tensor is copied for it.
"""
from __future__ import annotations

import operator
import warnings

import torch
import torch.fx as fx

from compiler import graph_replay, runtime

runtime.load()

_APPEND = torch.ops.b200.rope_append.default
_FUNCTIONAL = torch.ops.higher_order.auto_functionalized_v2
_PLAIN = ("q", "k", "v", "cos", "sin", "positions", "slots")
_CACHES = ("k_cache", "v_cache")
_ATTEND = torch.ops.b200.paged_attention.default
# Ops that take a cache and return nothing that aliases it.
_READERS = (_ATTEND, _APPEND)
_VIEWS = graph_replay._NO_LAUNCH | {operator.getitem}


def _caches_of(node: fx.Node):
    """The two base nodes of a functional append on whole tensors, else None."""
    if not (node.op == "call_function" and node.target == _FUNCTIONAL and node.args[:1] == (_APPEND,)):
        return None
    kw = node.kwargs
    if set(kw) != {*_PLAIN, "_all_bases", *(f"_{c}_base_index" for c in _CACHES)}:
        return None  # a cache is a view of its base: left functional
    where = [kw[f"_{c}_base_index"] for c in _CACHES]
    if not all(isinstance(i, int) for i in where) or where[0] == where[1] or len(kw["_all_bases"]) != 2:
        return None
    bases = [kw["_all_bases"][i] for i in where]
    if not all(isinstance(b, fx.Node) and b.op == "placeholder" for b in bases):
        return None
    return bases


def inplace_append(gm: fx.GraphModule) -> fx.GraphModule:
    order = {n: i for i, n in enumerate(gm.graph.nodes)}
    changed = False
    for node in list(gm.graph.nodes):
        bases = _caches_of(node)
        if bases is None:
            continue
        # Every other reader of the state before the append is done by then
        # and keeps no view of it.
        if any(u is not node and (order.get(u, 0) > order[node] or u.target not in _READERS)
               for b in bases for u in b.users):
            continue
        if any(u.target is not operator.getitem for u in node.users):
            continue
        with gm.graph.inserting_before(node):
            new = gm.graph.call_function(_APPEND, tuple(node.kwargs[n] for n in _PLAIN) + tuple(bases))
        order[new] = order[node]
        # results: the op's, then the bases' new states in the order of _all_bases
        results = [new] + list(node.kwargs["_all_bases"])
        val = node.meta.get("val")
        if isinstance(val, (tuple, list)):
            new.meta["val"] = val[0]
        for u in list(node.users):
            u.replace_all_uses_with(results[u.args[1]])
            gm.graph.erase_node(u)
        gm.graph.erase_node(node)
        changed = True
    if changed:
        gm.graph.lint()
        gm.recompile()
    left = sum(n.op == "call_function" and n.target == _FUNCTIONAL and n.args[:1] == (_APPEND,) for n in gm.graph.nodes)
    if left:
        warnings.warn(f"{left} b200::rope_append of a compiled graph copy the tensors that hold their caches, whole, at "
                      "every call: pass each cache as a tensor of its own, and attend over it behind the append")
    return gm


def appended_inputs(gm: fx.GraphModule) -> tuple:
    """Indices of the graph inputs that the graph appends to in place, if
    running the graph twice leaves what running it once does: every other use
    of them comes behind the append.  () when there is none, None when a
    graph that writes its inputs must not be run twice."""
    inputs = [n for n in gm.graph.nodes if n.op == "placeholder"]
    order = {n: i for i, n in enumerate(gm.graph.nodes)}
    found = set()
    for node in gm.graph.nodes:
        if node.op == "call_function" and node.target == _APPEND:
            for b in node.args[7:9]:
                if b not in inputs or any(order[u] < order[node] for u in b.users):
                    return None
                found.add(inputs.index(b))
    return tuple(sorted(found))


def attended_inputs(gm: fx.GraphModule) -> tuple:
    """Indices of the graph inputs that are caches and nothing else: the graph
    attends over them, or over views of them, and has no other use for them."""
    def cache_alone(n):
        return bool(n.users) and all(
            u.op == "call_function" and not u.kwargs
            and (u.target == _ATTEND and n in u.args[1:3] and n not in (u.args[0], *u.args[3:])
                 or u.target in _VIEWS and cache_alone(u))
            for u in n.users)

    return tuple(i for i, n in enumerate(n for n in gm.graph.nodes if n.op == "placeholder") if cache_alone(n))
