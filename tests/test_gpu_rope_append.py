"""b200::rope_append against the formula in 64 bits.

Bound of a rotated element: two fp32 products and a sum (3 * 2^-24 of the
products' magnitudes) and one rounding (half a step of the type).  Values,
unrotated columns and every place of the cache outside the appended slots
are bit-equal."""
import pytest
import torch

import serving_reference as ref
from compiler import runtime
from compiler.runtime import cabi

pytestmark = pytest.mark.gpu
runtime.load()


def make(t, H, hkv, D, R, page, dtype, seed=0, table=torch.float32, fused=True, index=torch.int64, reach=200):
    g = torch.Generator("cuda").manual_seed(seed + t + D)
    if fused:
        qkv = torch.randn(t, (H + 2 * hkv) * D, device="cuda", generator=g).to(dtype)
        q, k, v = (x.unflatten(1, (-1, D)) for x in qkv.split([H * D, hkv * D, hkv * D], 1))
    else:
        q, k, v = (torch.randn(t, h, D, device="cuda", generator=g).to(dtype) for h in (H, hkv, hkv))
    angle = torch.rand(reach, R // 2, device="cuda", generator=g) * 6.3
    cos, sin = angle.cos().to(table), angle.sin().to(table)
    pages = -(-t // page) + 2
    kc, vc = (torch.randn(pages, page, hkv, D, device="cuda", generator=g).to(dtype) for _ in range(2))
    pos = torch.randint(0, reach, (t,), device="cuda", generator=g).to(index)
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:t].to(index)
    return q, k, v, cos, sin, pos, slots, kc, vc


def check(before, q_out, args):
    q, k, v, cos, sin, pos, slots, kc, vc = args
    dt, R = q.dtype, 2 * cos.shape[1]
    h = ref.HALF_STEP[dt]

    def close(got, x):
        c, s = cos[pos.long().clamp(0, len(cos) - 1)], sin[pos.long().clamp(0, len(cos) - 1)]
        y, size = ref.rotate(x, c, s)
        tiny = 2.0**-25 if dt == torch.float16 else 0.0
        assert ((got.double() - y).abs() <= y.abs() * h * 1.001 + size * 3 * 2.0**-24 + tiny).all()
        assert torch.equal(got[..., R:], x[..., R:])

    close(q_out, q)
    live = slots >= 0
    at = slots.long()[live]
    close(kc.reshape(-1, *kc.shape[2:])[at], k[live])
    # pos of skipped tokens is not checked for keys
    assert torch.equal(vc.reshape(-1, *vc.shape[2:])[at], v[live])
    keep = torch.ones(kc.shape[0] * kc.shape[1], dtype=torch.bool, device="cuda")
    keep[at] = False
    for now, old in zip((kc, vc), before):
        assert torch.equal(now.reshape(-1, *now.shape[2:])[keep], old.reshape(-1, *old.shape[2:])[keep])


def run(args):
    before = args[7].clone(), args[8].clone()
    out = torch.ops.b200.rope_append(*args)
    q, k, v, cos, sin, pos, slots, kc, vc = args
    live = slots >= 0
    sub = (q, k[live], v[live])
    check(before, out, args) if live.all() else check_some(before, out, args)
    assert runtime.gemm_status() == 0
    return sub


def check_some(before, out, args):
    """With tokens that are not appended: queries all turned, the rest as check()."""
    q, k, v, cos, sin, pos, slots, kc, vc = args
    live = slots >= 0
    y, size = ref.rotate(q, cos[pos.long()], sin[pos.long()])
    assert ((out.double() - y).abs() <= y.abs() * ref.HALF_STEP[q.dtype] * 1.001 + size * 3 * 2.0**-24 + 2.0**-25).all()
    check(before, out[live], (q[live], k[live], v[live], cos, sin, pos[live], slots[live], kc, vc))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,H,hkv,D,R,page", [
    (1, 32, 8, 128, 128, 16), (1, 1, 1, 64, 64, 1), (7, 32, 8, 64, 64, 16), (33, 28, 4, 128, 64, 24),
    (5, 8, 1, 128, 32, 64), (3, 4, 2, 80, 80, 16), (9, 6, 3, 96, 96, 7), (4, 2, 2, 72, 36, 16), (6, 3, 1, 10, 6, 3),
    (2, 4, 4, 64, 0, 16), (1000, 32, 8, 128, 128, 16), (3000, 16, 16, 64, 32, 32), (5, 0, 2, 64, 64, 16)])
def test_against_the_formula(t, H, hkv, D, R, page, dtype):
    run(make(t, H, hkv, D, R, page, dtype))


@pytest.mark.parametrize("table", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("fused", [True, False])
def test_types_of_tables_and_indexes(table, index, fused):
    run(make(50, 8, 2, 64, 64, 16, torch.bfloat16, table=table, index=index, fused=fused))


def test_tokens_that_are_not_appended():
    args = make(40, 8, 2, 64, 64, 16, torch.bfloat16)
    args[6][::3] = -1
    run(args)


@pytest.mark.parametrize("layout", ["hnd", "pair", "odd"])
def test_cache_layouts(layout):
    q, k, v, cos, sin, pos, slots, kc, vc = make(40, 8, 2, 64, 64, 16, torch.bfloat16)
    if layout == "hnd":
        kc, vc = (c.transpose(1, 2).contiguous().transpose(1, 2) for c in (kc, vc))
    elif layout == "pair":
        both = torch.stack([kc, vc], 1)
        kc, vc = both[:, 0], both[:, 1]
    else:  # rows that are not 16-byte aligned
        kc, vc = (torch.nn.functional.pad(c, (1, 2))[..., 1:65] for c in (kc, vc))
    run((q, k, v, cos, sin, pos, slots, kc, vc))


def test_cache_offsets_past_32_bits():
    """Pages whose element offset is above 2^31 (a cache of 4.3 GB a side)."""
    D, hkv, page = 128, 8, 128
    pages = 2**31 // (page * hkv * D) + 4
    q, k, v, cos, sin, pos, _, _, _ = make(3, 8, hkv, D, D, page, torch.bfloat16)
    kc, vc = (torch.zeros(pages, page, hkv, D, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    slots = torch.tensor([pages * page - 1, 0, (pages - 3) * page + 5], device="cuda")
    torch.ops.b200.rope_append(q, k, v, cos, sin, pos, slots, kc, vc)
    flat = vc.view(-1, hkv, D)
    assert torch.equal(flat[slots], v)
    want, size = ref.rotate(k, cos[pos], sin[pos])
    assert ((kc.view(-1, hkv, D)[slots].double() - want).abs() <= want.abs() * 2.0**-8 * 1.001 + size * 1e-6).all()
    assert int((flat.view(-1, hkv * D).abs().amax(1) > 0).sum()) == 3


def test_an_index_out_of_range_is_reported_and_not_written():
    args = make(8, 4, 2, 64, 64, 16, torch.bfloat16)
    kc, vc = args[7], args[8]
    args[6][2] = kc.shape[0] * kc.shape[1]  # a slot past the cache
    args[5][4] = 10**6                      # a position past the tables
    before = kc.clone(), vc.clone()
    runtime.gemm_status()
    torch.ops.b200.rope_append(*args)
    with pytest.raises(RuntimeError, match="status 9"):
        runtime.check_status()
    runtime.check_status()
    good = torch.tensor([0, 1, 3, 5, 6, 7], device="cuda")
    flat = vc.view(-1, 2, 64)
    assert torch.equal(flat[args[6][good]], args[2][good])
    assert torch.equal(flat[args[6][4]], before[1].view(-1, 2, 64)[args[6][4]])


def test_refusals():
    q, k, v, cos, sin, pos, slots, kc, vc = make(8, 4, 2, 64, 64, 16, torch.bfloat16)
    op = torch.ops.b200.rope_append
    for bad in (lambda: op(q, k[:7], v[:7], cos, sin, pos, slots, kc, vc),
                lambda: op(q, k.half(), v, cos, sin, pos, slots, kc, vc),
                lambda: op(q, k, v, cos, sin, pos, slots, kc, vc[:1]),
                lambda: op(q, k, v, cos, sin, pos, slots, kc.half(), vc.half()),
                lambda: op(q, k, v, cos.half(), sin.half(), pos, slots, kc, vc),
                lambda: op(q, k, v, cos, sin, pos.float(), slots, kc, vc),
                lambda: op(q, k, v, cos, sin, pos, slots[:3], kc, vc),
                lambda: op(q, k, v, cos, sin, pos, slots.cpu(), kc, vc),
                lambda: op(q, k, v, cos, sin, pos, slots, kc[:, :, :1], vc[:, :, :1]),
                lambda: op(q, k, v, torch.cat([cos, cos], 1), torch.cat([sin, sin], 1), pos, slots, kc, vc),
                lambda: op(q, k, v, cos, sin, pos, slots, kc[:1].expand(4, 16, 2, 64), vc[:1].expand(4, 16, 2, 64)),
                lambda: op(q.float(), k.float(), v.float(), cos, sin, pos, slots, kc.float(), vc.float()),
                lambda: op(q.clone().requires_grad_(), k, v, cos, sin, pos, slots, kc, vc)):
        with pytest.raises(RuntimeError):
            bad()


def test_replayed_graph_appends_where_the_slots_say_now():
    args = make(16, 8, 2, 64, 64, 16, torch.bfloat16)
    q, k, v, cos, sin, pos, slots, kc, vc = args
    torch.ops.b200.rope_append(*args)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = torch.ops.b200.rope_append(*args)
    slots.copy_(torch.randperm(kc.shape[0] * kc.shape[1], device="cuda")[:16])
    pos.add_(3).remainder_(200)
    q.mul_(0.5)
    before = kc.clone(), vc.clone()
    g.replay()
    torch.cuda.synchronize()
    check(before, out, args)


def test_c_abi():
    args = make(20, 8, 2, 128, 128, 16, torch.float16)
    before = args[7].clone(), args[8].clone()
    out = torch.empty(20, 8, 128, device="cuda", dtype=torch.float16)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    cabi.rope_append(*args, out, status=status)
    assert status.item() == 0
    check(before, out, args)


def test_strides_of_dims_of_one_element_do_not_matter():
    q, k, v, cos, sin, pos, slots, kc, vc = make(1, 1, 1, 64, 64, 16, torch.bfloat16, fused=False)
    one = lambda t: t.as_strided(t.shape, tuple(s if n > 1 else 7 for n, s in zip(t.shape, t.stride())))  # noqa: E731
    run((one(q), one(k), one(v), cos, sin, pos, slots, one(kc), vc))
