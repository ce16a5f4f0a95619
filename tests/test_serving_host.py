"""CPU checks of the serving operators: what the C ABI refuses before any
launch, the ctypes layout, the registered schemas and fake implementations."""
import ctypes
import os
import subprocess

import pytest
import torch

from compiler import runtime
from compiler.runtime import cabi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INCLUDE = os.path.join(ROOT, "include")
runtime.load()

STRUCTS = {"B200kAddNormArgs": cabi.AddNormArgs, "B200kRopeAppendArgs": cabi.RopeAppendArgs,
           "B200kPagedAttentionArgs": cabi.PagedAttentionArgs}
OK, ARG, ALIGN, SHAPE, UNSUPPORTED, DEVICE = 0, 1, 2, 3, 4, 8


def test_ctypes_layout_matches_c(tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "b200k.h"', "int main(void) {"]
    for cname, cls in STRUCTS.items():
        lines.append(f'  printf("{cname} size %zu\\n", sizeof({cname}));')
        lines += [f'  printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in cls._fields_]
    lines.append('  printf("E4M3 E4M3 %d\\n", (int)B200K_E4M3); return 0; }')
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines))
    subprocess.run(["gcc", "-I", INCLUDE, str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines():
        cname, field, value = line.split()
        if cname == "E4M3":
            assert int(value) == cabi.E4M3
            continue
        cls = STRUCTS[cname]
        assert (ctypes.sizeof(cls) if field == "size" else getattr(cls, field).offset) == int(value), line


def test_status_string():
    assert cabi.library().b200k_status_string(9).decode().startswith("an index read on the device")


def norm_args(**kw):
    a = cabi.AddNormArgs()
    a.rows, a.cols, a.x, a.residual, a.sum, a.out = 4, 256, 4096, 8192, 12288, 16384
    a.x_row_stride = a.residual_row_stride = 256
    a.dtype = a.out_dtype = cabi.BF16
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(rows=0), OK), (dict(cols=0), OK), (dict(rows=-1), SHAPE), (dict(x=0), ARG), (dict(sum=0), ARG),
    (dict(out=0), ARG), (dict(dtype=cabi.F64, out_dtype=cabi.F64), UNSUPPORTED), (dict(out_dtype=cabi.F32), UNSUPPORTED),
    (dict(weight=4096, w_dtype=cabi.I32), UNSUPPORTED), (dict(flags=2), UNSUPPORTED), (dict(out_dtype=cabi.E4M3), ARG),
    (dict(out_dtype=cabi.E4M3, scale=4096, group=64), SHAPE),
    (dict(out_dtype=cabi.E4M3, scale=4096, group=128, cols=200), SHAPE), (dict(rows=1 << 31), SHAPE),
])
def test_add_rms_norm_refuses(kw, code):
    assert cabi.library().b200k_add_rms_norm(ctypes.byref(norm_args(**kw)), None) == code


def append_args(**kw):
    a = cabi.RopeAppendArgs()
    a.tokens, a.heads, a.kv_heads, a.head_dim, a.rot_dim, a.num_pages, a.page_size = 4, 8, 2, 64, 64, 10, 16
    a.q, a.k, a.v, a.q_out, a.k_cache, a.v_cache, a.cos, a.sin = range(4096, 4096 * 9, 4096)
    a.positions = a.slots = 4096
    a.table_rows, a.table_stride = 100, 32
    a.dtype, a.table_dtype, a.positions_dtype, a.slots_dtype = cabi.BF16, cabi.F32, cabi.I64, cabi.I64
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(tokens=0), OK), (dict(tokens=-1), SHAPE), (dict(q=0), ARG), (dict(v=0), ARG), (dict(k_cache=0), ARG),
    (dict(positions=0), ARG), (dict(slots=0), ARG), (dict(cos=0), ARG), (dict(table_rows=0), ARG),
    (dict(dtype=cabi.F32), UNSUPPORTED), (dict(table_dtype=cabi.F16), UNSUPPORTED),
    (dict(slots_dtype=cabi.F32), UNSUPPORTED), (dict(rot_dim=33), SHAPE), (dict(rot_dim=66), SHAPE),
    (dict(num_pages=1 << 30), SHAPE),
])
def test_rope_append_refuses(kw, code):
    assert cabi.library().b200k_rope_append(ctypes.byref(append_args(**kw)), None) == code


def attn_args(**kw):
    a = cabi.PagedAttentionArgs()
    a.tokens, a.seqs, a.heads, a.kv_heads, a.head_dim = 4, 2, 8, 2, 64
    a.num_pages, a.page_size, a.table_cols, a.table_stride = 10, 16, 4, 4
    a.q, a.k_cache, a.v_cache, a.out, a.page_table, a.q_start, a.kv_len = range(4096, 4096 * 8, 4096)
    a.q_strides[:] = [512, 64]
    a.cache_strides[:] = [16 * 128, 128, 64]
    a.dtype = cabi.BF16
    for k, v in kw.items():
        if isinstance(v, list):
            getattr(a, k)[:] = v
        else:
            setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(tokens=0), OK), (dict(tokens=-1), SHAPE), (dict(head_dim=96), UNSUPPORTED), (dict(kv_heads=3), SHAPE),
    (dict(kv_heads=0), SHAPE), (dict(q=0), ARG), (dict(dtype=cabi.F32), UNSUPPORTED), (dict(softcap=-1.0), ARG),
    (dict(window=-1), ARG), (dict(q=4098), ALIGN), (dict(q_strides=[510, 64]), ALIGN),
    (dict(cache_strides=[2048, 130, 64]), ALIGN), (dict(softcap=float("nan")), ARG),
    (dict(softcap=float("inf")), ARG), (dict(scale=float("inf")), ARG), (dict(scale=float("nan")), ARG),
])
def test_paged_attention_refuses(kw, code):
    assert cabi.library().b200k_paged_attention(ctypes.byref(attn_args(**kw)), None) == code


def test_workspace_query_refuses():
    lib, n = cabi.library(), ctypes.c_int64(-1)
    assert lib.b200k_paged_attention_workspace(None, ctypes.byref(n)) == ARG
    assert lib.b200k_paged_attention_workspace(ctypes.byref(attn_args(head_dim=80)), ctypes.byref(n)) == UNSUPPORTED
    assert lib.b200k_paged_attention_workspace(ctypes.byref(attn_args(tokens=0)), ctypes.byref(n)) == OK
    assert n.value == 0


def test_fakes_have_the_outputs_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x = torch.empty(3, 5, 256, device="cuda", dtype=torch.bfloat16)
        w = torch.empty(256, device="cuda", dtype=torch.bfloat16)
        out, total = torch.ops.b200.add_rms_norm(x, x, w, 1e-5)
        assert out.shape == total.shape == x.shape and out.dtype == x.dtype
        q8, scale, total = torch.ops.b200.add_rms_norm_quant(x, x, w, 1e-5, 128)
        assert q8.dtype == torch.float8_e4m3fn and scale.shape == (3, 5, 2) and scale.dtype == torch.float32
        assert torch.ops.b200.add_rms_norm_quant(x, x, w, 1e-5)[1].shape == (3, 5, 1)
        q = torch.empty(7, 8, 64, device="cuda", dtype=torch.float16)
        i = torch.empty(8, device="cuda", dtype=torch.int32)
        c = torch.empty(4, 16, 2, 64, device="cuda", dtype=torch.float16)
        assert torch.ops.b200.paged_attention(q, c, c, i.view(2, 4), i[:3], i[:2]).shape == q.shape
        assert torch.ops.b200.rope_append(q, q[:, :2], q[:, :2], i.view(2, 4).float(), i.view(2, 4).float(), i[:7],
                                          i[:7], c, c).shape == q.shape


def test_the_append_declares_what_it_writes():
    s = str(torch.ops.b200.rope_append.default._schema)
    assert "Tensor(a!) k_cache, Tensor(b!) v_cache" in s


@pytest.mark.parametrize("op", ["add_rms_norm", "add_rms_norm_quant", "rope_append", "paged_attention"])
def test_inputs_that_ask_for_a_gradient_are_refused_when_traced(op):
    """No gradient is defined: not only the kernels but a trace (on fake
    tensors) refuses, which would otherwise compile to a backward without the
    op's share."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    f = getattr(torch.ops.b200, op)
    with FakeTensorMode(allow_non_fake_inputs=True):
        def t(*shape, dtype=torch.bfloat16):
            return torch.empty(*shape, dtype=dtype, device="cuda")
        cache = t(4, 16, 2, 64), t(4, 16, 2, 64)
        ints = t(3, dtype=torch.int32)
        args = {"add_rms_norm": (t(3, 256), t(3, 256), None, 1e-5),
                "add_rms_norm_quant": (t(3, 256), t(3, 256), None, 1e-5, 128),
                "rope_append": (t(3, 8, 64), t(3, 2, 64), t(3, 2, 64), t(9, 32), t(9, 32), ints, ints, *cache),
                "paged_attention": (t(3, 8, 64), *cache, t(2, 4, dtype=torch.int32), ints, ints[:2])}[op]
        with torch.no_grad():
            f(*args)
        args[0].requires_grad_()
        with pytest.raises(RuntimeError, match="no gradient is defined"):
            f(*args)
        with torch.no_grad():
            f(*args)
