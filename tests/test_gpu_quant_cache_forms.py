"""Calls over e4m3 caches that the documentation allows: one scale for many rows by
strides of zero, inference mode, and slots that appear twice."""
import pytest
import torch

import quant_cache as qc
import quant_reference as quant
import serving_reference as ref
from compiler import runtime

pytestmark = pytest.mark.gpu
runtime.load()
ops = torch.ops.b200
BF = torch.bfloat16


@pytest.mark.parametrize("m", [1, 20, 100])
@pytest.mark.parametrize("shared", ["heads", "rows", "all"])
def test_expanded_scales(shared, m):
    """Scales of a head, of a row of all heads, of the whole cache."""
    q, k8, v8, ks, vs, *rest = qc.paged_inputs([m, 1], [150, 40], 8, 2, 64, 16, BF)
    one = {"heads": (1, 1, 2), "rows": (*ks.shape[:2], 1), "all": (1, 1, 1)}[shared]
    g = torch.Generator("cuda").manual_seed(0)
    ks, vs = (((1 + torch.rand(one, device="cuda", generator=g)) / 150).expand(ks.shape) for _ in range(2))
    x = (q, k8, v8, ks, vs, *rest)
    out = ops.paged_attention_quant(*x)
    qc.attention_close(out, x, ref.default_scale(64))
    assert torch.equal(out, ops.paged_attention_quant(q, k8, v8, ks.contiguous(), vs.contiguous(), *rest))


def test_inference_mode():
    with torch.inference_mode():
        q, k8, v8, ks, vs, *rest = qc.paged_inputs([1, 40], [150, 40], 8, 2, 64, 16, BF)
        x = (q, k8, v8, ks, vs, *rest)
        qc.attention_close(ops.paged_attention_quant(*x), x, ref.default_scale(64))
        k, v = (torch.randn(41, 2, 64, device="cuda").to(BF) for _ in range(2))
        none, at = torch.ones(1, 0, device="cuda"), torch.arange(41, device="cuda")
        k8.view(torch.uint8).zero_()
        assert torch.equal(ops.rope_append_quant(q, k, v, none, none, at * 0, at, k8, v8, ks, vs), q)
        back = qc.values(k8, ks)[:2].flatten(0, 1)[:32]
        assert ((back - k[:32].double()).abs() <= k[:32].double().abs().amax(-1, keepdim=True) * 2.0**-4).all()


def test_slots_that_appear_twice_stay_in_their_row():
    """Codes and scale of such a row are the tokens', in any mixture; every other row is as it would be."""
    T, KV, D = 64, 2, 64
    q, k, v = (torch.randn(T, h, D, device="cuda").to(BF) for h in (4, KV, KV))
    none = torch.ones(1, 0, device="cuda")
    slots = torch.arange(T, device="cuda")
    slots[40:] = 7
    caches = [torch.full((8, 16, KV, D), 0x55, device="cuda", dtype=torch.uint8).view(quant.E4M3) for _ in range(2)]
    scales = [torch.full((8, 16, KV), 3.0, device="cuda") for _ in range(2)]
    ops.rope_append_quant(q, k, v, none, none, slots * 0, slots, *caches, *scales)
    alone = [torch.full((8, 16, KV, D), 0x55, device="cuda", dtype=torch.uint8).view(quant.E4M3) for _ in range(2)]
    alone_s = [torch.full((8, 16, KV), 3.0, device="cuda") for _ in range(2)]
    ops.rope_append_quant(q[:40], k[:40], v[:40], none, none, slots[:40] * 0, slots[:40], *alone, *alone_s)
    other = torch.arange(128, device="cuda") != 7
    for a, b in zip((*caches, *scales), (*alone, *alone_s)):
        a, b = (t.view(torch.uint8) if t.dtype == quant.E4M3 else t for t in (a, b))
        assert torch.equal(a.flatten(0, 1)[other], b.flatten(0, 1)[other])
    assert runtime.gemm_status() == 0
