"""b200::rope_append_quant against the formula in 64 bits.

Bounds.  q: as b200::rope_append's (test_gpu_rope_append.py).  A cached row is
rotated in fp32, 3 * 2^-24 of the products' magnitudes off, at most R of the
row's largest; its scale has two roundings more (2^-23); a code is half a step
of e4m3 off, plus what the row's error is over the scale (and 2^-22 relative
of the quotient).  Every place of the caches and scales outside the appended
slots is bit-equal."""
import pytest
import torch

import quant_cache as qc
import quant_reference as quant
import serving_reference as ref
from compiler import runtime
from compiler.runtime import cabi
from test_gpu_rope_append import make as make16

pytestmark = pytest.mark.gpu
runtime.load()
op = torch.ops.b200.rope_append_quant


def make(*args, order="phs", **kw):
    *rest, kc, vc = make16(*args, **kw)
    (k8, ks), (v8, vs) = qc.quantised(kc, order), qc.quantised(vc, order)
    return (*rest, k8, v8, ks, vs)


def raw(t):
    return t.view(torch.uint8) if t.dtype == quant.E4M3 else t


def copies(args):
    return [t.clone() for t in args[7:]]


def check(before, q_out, args):
    q, k, v, cos, sin, pos, slots, k8, v8, ks, vs = args
    dt, R = q.dtype, 2 * cos.shape[1]
    y, size = ref.rotate(q, cos[pos.long()], sin[pos.long()])
    tiny = 2.0**-25 if dt == torch.float16 else 0.0
    assert ((q_out.double() - y).abs() <= y.abs() * ref.HALF_STEP[dt] * 1.001 + size * 3 * 2.0**-24 + tiny).all()
    assert torch.equal(q_out[..., R:], q[..., R:])
    live = slots >= 0
    page = k8.shape[1]
    at = slots.long()[live] // page, slots.long()[live] % page
    turned, size = ref.rotate(k[live], cos[pos.long()[live]], sin[pos.long()[live]])
    for codes, scale, row, off in ((k8, ks, turned, size * 3 * 2.0**-24), (v8, vs, v[live].double(), turned * 0)):
        top = row.abs().amax(-1).clamp_min(quant.MIN_AMAX) / quant.MAX
        s = scale[at].double()
        assert ((s - top).abs() <= top * 2.0**-22 + off.amax(-1) / quant.MAX).all()
        z, err = row / s[..., None], off / s[..., None]
        got = codes.view(torch.uint8)[at].view(quant.E4M3).double()
        assert ((got - z).abs() <= quant.code_step(z) + err + z.abs() * 2.0**-22).all()
    keep = torch.ones(k8.shape[:2], dtype=torch.bool, device="cuda")
    keep[at] = False
    for now, old in zip(args[7:], before):
        same = raw(now) == raw(old)
        assert (same if same.dim() == 3 else same.all(-1))[keep].all()


def run(args):
    before = copies(args)
    check(before, op(*args), args)
    assert runtime.gemm_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,H,hkv,D,R,page", [
    (1, 32, 8, 128, 128, 16), (1, 1, 1, 64, 64, 1), (7, 32, 8, 64, 64, 16), (33, 28, 4, 128, 64, 24), (5, 8, 1, 128, 32, 64),
    (3, 4, 2, 80, 80, 16), (9, 6, 3, 96, 96, 7), (4, 2, 2, 72, 36, 16), (6, 3, 1, 10, 6, 3), (2, 4, 4, 64, 0, 16), (6, 2, 1, 16, 16, 4),
    (5, 2, 2, 512, 256, 4), (3, 1, 1, 1024, 64, 2), (1000, 32, 8, 128, 128, 16), (3000, 16, 16, 64, 32, 32), (5, 0, 2, 64, 64, 16)])
def test_against_the_formula(t, H, hkv, D, R, page, dtype):
    run(make(t, H, hkv, D, R, page, dtype))


@pytest.mark.parametrize("table", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("fused", [True, False])
def test_types_of_tables_and_indexes(table, index, fused):
    run(make(50, 8, 2, 64, 64, 16, torch.bfloat16, table=table, index=index, fused=fused))


@pytest.mark.parametrize("t", [40, 3000])
def test_tokens_that_are_not_appended(t):
    args = make(t, 8, 2, 64, 64, 16, torch.bfloat16)
    args[6][::3] = -1
    run(args)


@pytest.mark.parametrize("order", ["psh", "phs", "hps"])
@pytest.mark.parametrize("layout", ["hnd", "pair", "odd"])
def test_cache_and_scale_layouts(layout, order):
    *rest, k8, v8, ks, vs = make(40, 8, 2, 64, 64, 16, torch.bfloat16, order=order)
    if layout == "hnd":
        k8, v8 = (c.view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(quant.E4M3) for c in (k8, v8))
    elif layout == "pair":
        both = torch.stack([raw(k8), raw(v8)], 1).view(quant.E4M3)
        k8, v8 = both[:, 0], both[:, 1]
        both = torch.stack([ks, vs], 1)
        ks, vs = both[:, 0], both[:, 1]
    else:  # rows that are not 8-byte aligned
        k8, v8 = (torch.nn.functional.pad(raw(c), (1, 2))[..., 1:65].view(quant.E4M3) for c in (k8, v8))
    run((*rest, k8, v8, ks, vs))


def test_rows_of_zeros_infinities_and_nan():
    args = make(6, 4, 2, 64, 64, 16, torch.bfloat16)
    k, v, slots, k8, v8, ks, vs = args[1], args[2], args[6], *args[7:]
    k[0], v[0] = 0, 0
    v[1, 0, 3], v[2, 1, 5] = float("nan"), float("inf")
    k[3, 0, 7] = float("nan")
    op(*args)
    at = slots // 16, slots % 16
    small = torch.tensor(1e-12 / 448, dtype=torch.float32, device="cuda")
    kr, vr = (c.view(torch.uint8)[at].view(quant.E4M3).float() for c in (k8, v8))
    assert (kr[0] == 0).all() and (vr[0] == 0).all()
    assert ((ks[at][0] - small).abs() <= small * 2.0**-22).all() and ((vs[at][0] - small).abs() <= small * 2.0**-22).all()
    assert vr[1, 0].isnan().all() and vs[at][1, 0].isnan() and vr[1, 1].isfinite().all()
    assert vr[2, 1, 5].isnan() and vs[at][2, 1].isinf() and (vr[2, 1, :5] == 0).all()
    assert kr[3, 0].isnan().all() and ks[at][3, 0].isnan() and kr[3, 1].isfinite().all()


def test_cache_offsets_past_32_bits():
    """Pages whose offset is above 2^31 (a cache of 2.1 GB a side)."""
    D, hkv, page = 128, 8, 128
    pages = 2**31 // (page * hkv * D) + 4
    q, k, v, cos, sin, pos, *_ = make16(3, 8, hkv, D, D, page, torch.bfloat16)
    k8, v8 = (torch.zeros(pages, page, hkv, D, device="cuda", dtype=torch.uint8).view(quant.E4M3) for _ in range(2))
    ks, vs = (torch.zeros(pages, page, hkv, device="cuda") for _ in range(2))
    slots = torch.tensor([pages * page - 1, 0, (pages - 3) * page + 5], device="cuda")
    op(q, k, v, cos, sin, pos, slots, k8, v8, ks, vs)
    got = v8.view(torch.uint8).view(-1, hkv, D)[slots].view(quant.E4M3)
    z = v.double() / vs.view(-1, hkv)[slots].double()[..., None]
    assert ((got.double() - z).abs() <= quant.code_step(z) + z.abs() * 2.0**-22).all()
    assert int((vs.view(-1, hkv).amax(1) > 0).sum()) == 3 and int((ks.view(-1, hkv).amax(1) > 0).sum()) == 3


def test_an_index_out_of_range_is_reported_and_not_written():
    args = make(8, 4, 2, 64, 64, 16, torch.bfloat16)
    k8, slots = args[7], args[6]
    slots[2] = k8.shape[0] * k8.shape[1]  # a slot past the cache
    args[5][4] = 10**6                    # a position past the tables
    before = copies(args)
    runtime.gemm_status()
    op(*args)
    with pytest.raises(RuntimeError, match="status 9"):
        runtime.check_status()
    runtime.check_status()
    changed = (raw(args[8]) != raw(before[1])).flatten(0, 1).flatten(1).any(1)
    want = torch.zeros_like(changed)
    want[slots[torch.tensor([0, 1, 3, 5, 6, 7], device="cuda")]] = True
    assert torch.equal(changed, want)


def test_refusals():
    q, k, v, cos, sin, pos, slots, k8, v8, ks, vs = make(8, 4, 2, 64, 64, 16, torch.bfloat16)
    for bad in (lambda: op(q, k[:7], v[:7], cos, sin, pos, slots, k8, v8, ks, vs),
                lambda: op(q, k, v, cos, sin, pos, slots, k8.float().to(q.dtype), v8.float().to(q.dtype), ks, vs),
                lambda: op(q, k, v, cos, sin, pos, slots, k8.view(torch.uint8), v8.view(torch.uint8), ks, vs),
                lambda: op(q, k, v, cos, sin, pos, slots, k8, v8, ks[:1], vs[:1]),
                lambda: op(q, k, v, cos, sin, pos, slots, k8, v8, ks, vs.contiguous()),
                lambda: op(q, k, v, cos, sin, pos, slots, k8, v8, ks.double(), vs.double()),
                lambda: op(q, k, v, cos, sin, pos, slots, k8, v8, ks.cpu(), vs.cpu()),
                lambda: op(q, k, v, cos, sin, pos, slots, k8, k8, ks, vs),
                lambda: op(q, k, v, cos, sin, pos, slots, k8, v8, ks, ks),
                lambda: op(q, k, v, cos, sin, pos, slots, k8, v8, ks[:1].expand(ks.shape), vs[:1].expand(vs.shape)),
                lambda: op(q.clone().requires_grad_(), k, v, cos, sin, pos, slots, k8, v8, ks, vs)):
        with pytest.raises(RuntimeError):
            bad()


def test_replayed_graph_appends_where_the_slots_say_now():
    args = make(16, 8, 2, 64, 64, 16, torch.bfloat16)
    q, _, _, _, _, pos, slots, k8, *_ = args
    op(*args)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = op(*args)
    slots.copy_(torch.randperm(k8.shape[0] * k8.shape[1], device="cuda")[:16])
    pos.add_(3).remainder_(200)
    q.mul_(0.5)
    before = copies(args)
    g.replay()
    torch.cuda.synchronize()
    check(before, out, args)


def test_c_abi():
    args = make(20, 8, 2, 128, 128, 16, torch.float16)
    before = copies(args)
    out = torch.empty(20, 8, 128, device="cuda", dtype=torch.float16)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    cabi.rope_append_quant(*args, out, status=status)
    assert status.item() == 0
    check(before, out, args)
