"""torch.compile backend entry points (same API as the reference's
compiler/backend.py:1-24).

    from compiler.backend import custom_backend      # or `backend`
    model = torch.compile(model, backend=custom_backend)

``compiler(gm, example_inputs)`` is the AOTAutograd forward/backward compiler:
it runs the FX passes over the ATen graph and returns a boxed callable.  The
passes replace matched groups with calls of ``torch.ops.b200.*``, which launch
the hand-written sm_100a kernels of libb200k.so on the current stream.
"""
from __future__ import annotations

import torch
import torch.fx as fx
from torch._decomp import get_decompositions
from torch._dynamo.backends.common import aot_autograd
from torch._functorch.aot_autograd import make_boxed_func

from compiler import graph_replay, runtime
from compiler.optimization import config
from compiler.optimization.cat_inputs import contiguous_cat_inputs
from compiler.optimization.fusion_attention import fuse_attention
from compiler.optimization.fusion_epilogue import fuse_epilogue
from compiler.optimization.fusion_patchify import fuse_patchify
from compiler.optimization.fusion_pointwise import fuse_pointwise
from compiler.optimization.fusion_rope import fuse_gemm_rope, fuse_rope
from compiler.optimization.fusion_rowreduce import fuse_rowreduce
from compiler.optimization.inplace_append import appended_inputs, attended_inputs, inplace_append

runtime.load()


def _dump(gm: fx.GraphModule) -> None:
    print(gm.code)
    for n in gm.graph.nodes:
        if "b200_kernel" in n.meta:
            print(f"# {n.meta['b200_kernel']}: {' -> '.join(n.meta.get('b200_group', []))}")
            if "b200_program" in n.meta:
                print(f"#   program: {n.meta['b200_program']}")


# Graphs this process has compiled through the backend, and the fused GEMM
# nodes in them (diagnostic counts: callers check that their calls really
# went through the backend and its GEMM kernels).
GRAPHS_COMPILED = 0
GEMMS_FUSED = 0


def _passes(gm: fx.GraphModule) -> fx.GraphModule:
    global GRAPHS_COMPILED, GEMMS_FUSED
    GRAPHS_COMPILED += 1
    if config.EXTENSIONS:
        gm = inplace_append(gm)  # cache appends write their caches, not copies (extension)
    if config.EXTENSIONS and config.ENABLE_PATCHIFY:
        gm = fuse_patchify(gm)  # patch-embedding convolutions -> im2col + addmm (extension)
    if config.EXTENSIONS:
        gm = contiguous_cat_inputs(gm)  # broadcast cat inputs made contiguous (extension)
    if config.EXTENSIONS and config.ENABLE_ROWREDUCE:
        gm = fuse_rowreduce(gm)  # whole row groups (extension; runs first so the
        #                          pointwise passes do not split them)
    if config.EXTENSIONS and config.ENABLE_ATTENTION:
        gm = fuse_attention(gm)  # SDPA nodes -> the tcgen05 attention kernel (extension)
    if config.EXTENSIONS and config.ENABLE_ROPE:
        gm = fuse_rope(gm)  # x*cos + rotate_half(x)*sin (extension; before the
        #                     pointwise pass would take its multiply-add)
        if config.ENABLE_GEMM_ROPE:
            gm = fuse_gemm_rope(gm)  # a rotated q / k projection -> one GEMM (extension)
    if config.ENABLE_EPILOGUE:
        gm = fuse_epilogue(gm)  # pointwise groups that consume a matmul
    if config.ENABLE_POINTWISE:
        gm = fuse_pointwise(gm)  # the remaining pointwise groups
    GEMMS_FUSED += sum(1 for n in gm.graph.nodes
                       if n.op == "call_function" and n.target == torch.ops.b200.gemm_epilogue.default)
    if config.DUMP:
        _dump(gm)
    return gm


class StatusChecked:
    """Boxed callable around a compiled graph that launches GEMMs or the paged
    cache's kernels: before each call it raises if an earlier one on the
    device reported a device-side timeout or an index out of range, and after the call it queues an asynchronous read-back of the
    device's status word (``torch.ops.b200.status_check``).  Without it a
    timed-out GEMM would hand a partly written tensor to the rest of the
    graph with no error; with it the error surfaces at the next compiled
    call (or at ``runtime.check_status()``, which synchronises)."""

    def __init__(self, fn, device: int):
        self.fn = fn
        self.device = device
        # AOTAutograd's marker for the list-argument calling convention, on
        # the instance: the backward graph's callable reaches AOTAutograd
        # through a functools.wraps wrapper, which copies the instance's
        # __dict__ but not class attributes.
        self._boxed_call = True

    def __call__(self, args):
        torch.ops.b200.status_check(self.device, False)
        out = self.fn(args)
        torch.ops.b200.status_check(self.device, True)
        return out


# Ops whose kernels report through the device's status word: waits that run
# out, indexes out of range.
_REPORTING = (torch.ops.b200.gemm_epilogue.default, torch.ops.b200.rope_append.default,
              torch.ops.b200.paged_attention.default)


def _gemm_device(gm: fx.GraphModule, example_inputs) -> int | None:
    """CUDA device index of the graph's GEMM launches (and other launches that
    report through the status word), None when it has none."""
    for n in gm.graph.nodes:
        if n.op == "call_function" and n.target in _REPORTING:
            val = n.args[0].meta.get("val") if isinstance(n.args[0], fx.Node) else None
            if isinstance(val, torch.Tensor) and val.is_cuda:
                return val.device.index if val.device.index is not None else torch.cuda.current_device()
            for t in example_inputs:
                if isinstance(t, torch.Tensor) and t.is_cuda:
                    return t.device.index if t.device.index is not None else torch.cuda.current_device()
    return None


def _checked(gm: fx.GraphModule, example_inputs, fn):
    dev = _gemm_device(gm, example_inputs)
    return fn if dev is None else StatusChecked(fn, dev)


def compiler(gm: fx.GraphModule, example_inputs):
    """Forward and backward graphs of training: the passes, run op by op."""
    gm = _passes(gm)
    return _checked(gm, example_inputs, make_boxed_func(gm.forward))


def inference_compiler(gm: fx.GraphModule, example_inputs):
    """Inference graphs (no input requires grad): the passes, then CUDA-graph
    replay when the graph launches enough kernels (compiler/graph_replay.py;
    an extension, B200_CUDA_GRAPHS=0 turns it off)."""
    gm = _passes(gm)
    fn = make_boxed_func(gm.forward)
    if config.EXTENSIONS:
        caches = appended_inputs(gm)
        if caches is not None:
            fn = graph_replay.wrap(gm, fn, _static_inputs(), caches, attended_inputs(gm))
    return _checked(gm, example_inputs, fn)


def _static_inputs() -> tuple:
    """Indices of the graph inputs AOTAutograd marks static (the module's
    parameters and buffers, lifted to inputs by dynamo); () outside a
    dynamo compile."""
    ctx = torch._guards.TracingContext.try_get()
    meta = getattr(ctx, "fw_metadata", None) if ctx is not None else None
    return tuple(getattr(meta, "static_input_indices", None) or ())


custom_backend = aot_autograd(
    fw_compiler=compiler,
    bw_compiler=compiler,
    inference_compiler=inference_compiler,
    decompositions=get_decompositions([torch.ops.aten.gelu, torch.ops.aten.silu]),
)

# The reference's task statement calls the entry `backend`; both names work.
backend = custom_backend
