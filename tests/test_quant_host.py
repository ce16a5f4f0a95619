"""CPU checks of the 8-bit operators: what the C ABI refuses before any launch,
the ctypes layout, schemas and fake implementations, and the refusal of inputs
that ask for a derivative."""
import ctypes
import os
import subprocess

import pytest
import torch
from torch.autograd import forward_ad

from compiler import runtime
from compiler.runtime import cabi
from test_serving_host import ALIGN, ARG, INCLUDE, OK, SHAPE, UNSUPPORTED, append_args, attn_args

runtime.load()
E4M3 = torch.float8_e4m3fn
STRUCTS = {"B200kQuantGroupsArgs": cabi.QuantGroupsArgs, "B200kScaledMmArgs": cabi.ScaledMmArgs,
           "B200kRopeAppendQuantArgs": cabi.RopeAppendQuantArgs,
           "B200kPagedAttentionQuantArgs": cabi.PagedAttentionQuantArgs}


def test_ctypes_layout_matches_c(tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "b200k.h"', "int main(void) {"]
    for cname, cls in STRUCTS.items():
        lines.append(f'  printf("{cname} size %zu\\n", sizeof({cname}));')
        lines += [f'  printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in cls._fields_]
    lines.append("  return 0; }")
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines))
    subprocess.run(["gcc", "-I", os.path.abspath(INCLUDE), str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines():
        cname, field, value = line.split()
        cls = STRUCTS[cname]
        assert (ctypes.sizeof(cls) if field == "size" else getattr(cls, field).offset) == int(value), line


def fill(a, kw):
    for k, v in kw.items():
        if isinstance(v, list):
            getattr(a, k)[:] = v
        else:
            setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(rows=0), OK), (dict(cols=0), OK), (dict(rows=-1), SHAPE), (dict(cols=1 << 31), SHAPE), (dict(x=0), ARG),
    (dict(out=0), ARG), (dict(scale=0), ARG), (dict(dtype=cabi.F64), UNSUPPORTED), (dict(dtype=cabi.E4M3), UNSUPPORTED),
    (dict(x_row_stride=-1), SHAPE), (dict(rows=1 << 60), SHAPE),
])
def test_quant_groups_refuses(kw, code):
    a = cabi.QuantGroupsArgs()
    a.rows, a.cols, a.x, a.out, a.scale, a.x_row_stride, a.dtype = 4, 256, 4096, 8192, 12288, 256, cabi.BF16
    assert cabi.library().b200k_quant_groups(ctypes.byref(fill(a, kw)), None) == code
    assert cabi.library().b200k_quant_groups(None, None) == ARG


@pytest.mark.parametrize("kw,code", [
    (dict(M=0), OK), (dict(N=0), OK), (dict(M=-1), SHAPE), (dict(K=1 << 31), SHAPE), (dict(a=0), ARG), (dict(b=0), ARG),
    (dict(a_scale=0), ARG), (dict(b_scale=0), ARG), (dict(out=0), ARG), (dict(out_dtype=cabi.F64), UNSUPPORTED),
    (dict(out_dtype=cabi.E4M3), UNSUPPORTED), (dict(a=4097), ALIGN), (dict(b=4104), ALIGN), (dict(out=4098), ALIGN),
    (dict(a_stride_m=264), ALIGN), (dict(b_stride_n=128), ALIGN), (dict(tile=2), ARG), (dict(tile=-1), ARG),
    (dict(split=9), ARG), (dict(split=-1), ARG),
])
def test_scaled_mm_refuses(kw, code):
    a = cabi.ScaledMmArgs()
    a.M, a.N, a.K = 4, 8, 256
    a.a, a.b, a.a_scale, a.b_scale, a.out = range(4096, 4096 * 6, 4096)
    a.a_stride_m = a.b_stride_n = 256
    a.a_scale_strides[:], a.b_scale_strides[:] = [2, 1], [1, 1]
    a.out_dtype = cabi.BF16
    assert cabi.library().b200k_scaled_mm(ctypes.byref(fill(a, kw)), None) == code
    assert cabi.library().b200k_scaled_mm(None, None) == ARG


def with_scales(cls, base, kw):
    a = cls()
    a.base, a.k_scale, a.v_scale = base, 4096, 8192
    a.scale_strides[:] = [32, 2, 1]
    return fill(a, kw)


@pytest.mark.parametrize("base,kw,code", [
    (dict(tokens=0), {}, OK), (dict(q=0), {}, ARG), ({}, dict(k_scale=0), ARG), ({}, dict(v_scale=0), ARG),
    (dict(dtype=cabi.F32), {}, UNSUPPORTED), (dict(rot_dim=66), {}, SHAPE),
])
def test_rope_append_quant_refuses(base, kw, code):
    a = with_scales(cabi.RopeAppendQuantArgs, append_args(**base), kw)
    assert cabi.library().b200k_rope_append_quant(ctypes.byref(a), None) == code
    assert cabi.library().b200k_rope_append_quant(None, None) == ARG


@pytest.mark.parametrize("base,code", [
    (dict(tokens=0), OK), (dict(head_dim=96), UNSUPPORTED), (dict(kv_heads=3), SHAPE), (dict(q=0), ARG),
    (dict(dtype=cabi.E4M3), UNSUPPORTED), (dict(softcap=-1.0), ARG), (dict(cache_strides=[2048, 136, 64]), ALIGN),
    (dict(k_cache=4100), ALIGN), (dict(scale=float("nan")), ARG),
])
def test_paged_attention_quant_refuses(base, code):
    a = with_scales(cabi.PagedAttentionQuantArgs, attn_args(**base), {})
    assert cabi.library().b200k_paged_attention_quant(ctypes.byref(a), None) == code
    lib, n = cabi.library(), ctypes.c_int64(-1)
    assert lib.b200k_paged_attention_quant(None, None) == ARG
    assert lib.b200k_paged_attention_quant_workspace(None, ctypes.byref(n)) == ARG


def calls():
    """Per operator: arguments, and which of them are floating tensors."""
    def t(*shape, dtype=torch.bfloat16):
        return torch.empty(*shape, dtype=dtype, device="cuda")
    f32, i32 = torch.float32, torch.int32
    cache = t(4, 16, 2, 64, dtype=E4M3), t(4, 16, 2, 64, dtype=E4M3)
    scales = t(4, 16, 2, dtype=f32), t(4, 16, 2, dtype=f32)
    ints = t(3, dtype=i32)
    return {"quant_groups": ((t(3, 256),), [0]),
            "scaled_mm": ((t(3, 256, dtype=E4M3), t(64, 256, dtype=E4M3).t(), t(3, 2, dtype=f32), t(2, 1, dtype=f32),
                           torch.bfloat16), [2, 3]),
            "rope_append_quant": ((t(3, 8, 64), t(3, 2, 64), t(3, 2, 64), t(9, 32), t(9, 32), ints, ints, *cache, *scales),
                                  [0, 1, 2, 3, 4, 9, 10]),
            "paged_attention_quant": ((t(3, 8, 64), *cache, *scales, t(2, 4, dtype=i32), ints, ints[:2]), [0, 3, 4])}


OPS = ["quant_groups", "scaled_mm", "rope_append_quant", "paged_attention_quant"]


@pytest.mark.parametrize("op", OPS)
def test_inputs_that_ask_for_a_derivative_are_refused_when_traced(op):
    from torch._subclasses.fake_tensor import FakeTensorMode

    f = getattr(torch.ops.b200, op)
    with FakeTensorMode(allow_non_fake_inputs=True):
        for at in calls()[op][1]:
            args = list(calls()[op][0])
            with torch.no_grad():
                f(*args)
            args[at].requires_grad_()
            with pytest.raises(RuntimeError, match="no gradient is defined"):
                f(*args)
            with torch.no_grad():
                f(*args)
        with forward_ad.dual_level(), torch.no_grad():
            for at in calls()[op][1]:
                args = list(calls()[op][0])
                args[at] = forward_ad.make_dual(args[at], torch.ones_like(args[at]))
                with pytest.raises(RuntimeError, match="no gradient is defined"):
                    f(*args)


def test_fakes_have_the_outputs_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    ops = torch.ops.b200
    with FakeTensorMode():
        x = torch.empty(3, 5, 400, device="cuda", dtype=torch.bfloat16)
        out, scale = ops.quant_groups(x)
        assert out.shape == x.shape and out.dtype == E4M3 and scale.shape == (3, 5, 4) and scale.dtype == torch.float32
        out, scale = ops.quant_groups(x, True)
        assert out.shape == (3, 5, 200) and scale.shape == (3, 5, 2)
        c = {op: f(*args) for op, (args, _) in calls().items() if (f := getattr(ops, op))}
        assert c["scaled_mm"].shape == (3, 64) and c["scaled_mm"].dtype == torch.bfloat16
        assert c["rope_append_quant"].shape == c["paged_attention_quant"].shape == (3, 8, 64)


def test_the_append_declares_what_it_writes():
    s = str(torch.ops.b200.rope_append_quant.default._schema)
    assert "Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) k_scale, Tensor(d!) v_scale" in s
