"""b200::paged_attention_quant against the formula in 64 bits on what the
caches' codes and scales stand for (quant_cache.attention_close; the bound is
derived at serving_reference.attention_close: weights are rounded to f16 here,
whose half step is below bf16's).  Everything of the caches and scales that no
query may see holds NaN, and tables name no page that is not needed."""
import pytest
import torch

import quant_cache as qc
import quant_reference as quant
import serving_reference as ref
from compiler import runtime
from compiler.runtime import cabi

pytestmark = pytest.mark.gpu
runtime.load()
BF, HF = torch.bfloat16, torch.float16
op = torch.ops.b200.paged_attention_quant


def run(inputs, softcap=0.0, window=0, max_q=0, scale=0.0):
    q = inputs[0]
    runtime.gemm_status()
    out = op(*inputs, scale, softcap, window, max_q)
    qc.attention_close(out, inputs, scale or ref.default_scale(q.shape[2]), softcap, window)
    end = int(inputs[6][-1])
    assert out[end:].abs().sum() == 0
    assert runtime.gemm_status() == 0
    return out


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,hkv", [(32, 8), (8, 8), (8, 1), (7, 1), (28, 4), (40, 1), (6, 2)])
def test_single_tokens(H, hkv, D, dtype):
    ns = [1, 2, 15, 16, 17, 31, 32, 33, 100, 333, 1, 64]
    run(qc.paged_inputs([1] * len(ns), ns, H, hkv, D, 16, dtype))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,hkv,q", [(32, 8, 1), (8, 8, 1), (8, 1, 1), (7, 1, 1), (28, 4, 1), (8, 8, 5), (16, 8, 4), (16, 16, 8)])
def test_units_of_eight_rows(H, hkv, q, D, dtype):
    """Calls whose longest sequence is said to have at most 8 query rows; and a hint that is too small."""
    ns = [1, 31, 32, 33, 64, 700, 5, 2000, 0, 130]
    qs = [min(q, max(1, n)) for n in ns]
    run(qc.paged_inputs(qs, ns, H, hkv, D, 16, dtype, pad=2), max_q=q)
    qs[3], qs[5] = 20, 40
    run(qc.paged_inputs(qs, ns, H, hkv, D, 16, dtype, spread=4), max_q=q)
    run(qc.paged_inputs(qs, ns, H, hkv, D, 24, dtype, window=50), softcap=20.0, window=50, max_q=q)


@pytest.mark.parametrize("max_q", [0, 1])
@pytest.mark.parametrize("what", ["k", "v_scale"])
def test_a_nan_in_units_of_eight_rows(what, max_q):
    q, k8, v8, ks, vs, table, q_start, kv_len = qc.paged_inputs([1, 1], [200, 90], 8, 2, 128, 16, BF)
    clean = op(q, k8, v8, ks, vs, table, q_start, kv_len, 0.0, 0.0, 0, max_q)
    if what == "k":
        k8.view(torch.uint8)[table[0, 3].long(), 5, 1, 7] = 0x7F
    else:
        vs[table[0, 3].long(), 5, 1] = float("nan")
    out = op(q, k8, v8, ks, vs, table, q_start, kv_len, 0.0, 0.0, 0, max_q)
    assert out[0, 4:].isnan().all() and torch.equal(out[0, :4], clean[0, :4]) and torch.equal(out[1], clean[1])


@pytest.mark.parametrize("m", [1, 100])
@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 64, 100, 128])
def test_page_sizes(page, m):
    ns = [1, page, page + 1, 200, 3 * page - 1, 77]
    ns = [max(1, n) for n in ns]
    run(qc.paged_inputs([m] * len(ns), ns, 8, 2, 64, page, BF))
    run(qc.paged_inputs([m] * len(ns), ns, 4, 2, 128, page, BF))


@pytest.mark.parametrize("m", [1, 80])
@pytest.mark.parametrize("order", ["psh", "phs", "hps"])
@pytest.mark.parametrize("layout", ["nhd", "hnd", "pair"])
@pytest.mark.parametrize("D", [64, 128])
def test_cache_and_scale_layouts(layout, D, order, m):
    run(qc.paged_inputs([m, 4, 1], [100, 50, 7], 8, 2, D, 16, BF, layout=layout, order=order))


@pytest.mark.parametrize("softcap,window", [(30.0, 0), (5.0, 0), (0.0, 1), (0.0, 17), (0.0, 100), (50.0, 33), (1000.0, 0),
                                            (0.0, 10**6)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_caps_and_windows(softcap, window, D, dtype):
    qs, ns = [1, 3, 1, 8, 20], [90, 200, 5, 8, 300]
    run(qc.paged_inputs(qs, ns, 8, 2, D, 16, dtype, window=window), softcap, window)


@pytest.mark.parametrize("max_q", [0, 1, 33])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
def test_ragged_queries_and_rows_without_keys(D, dtype, max_q):
    qs = [0, 1, 3, 33, 5, 4, 0, 2]
    ns = [10, 40, 0, 33, 200, 2, 0, 2]
    out = run(qc.paged_inputs(qs, ns, 8, 2, D, 16, dtype, pad=5), max_q=max_q)
    assert out[1:4].abs().sum() == 0                       # kv_len 0
    start = sum(qs[:5])
    assert out[start:start + 2].abs().sum() == 0           # positions before the first key
    assert out[start + 2:start + 4].abs().sum() > 0


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("spread", [3, 12])
@pytest.mark.parametrize("m", [1, 7, 90])
def test_value_scales_far_apart(m, spread, dtype, D):
    run(qc.paged_inputs([m, 1], [300, 77], 8, 2, D, 16, dtype, spread=spread))


@pytest.mark.parametrize("dtype", [HF, BF])
@pytest.mark.parametrize("m", [1, 5, 100])  # rows, two row blocks, tiles
@pytest.mark.parametrize("sink", [0, 130])
@pytest.mark.parametrize("nats", [9.0, 13.0, 18.0])
@pytest.mark.parametrize("D", [64, 128])
def test_a_key_far_above_the_others(D, nats, sink, m, dtype):
    """... whose value is zero, with the scale of a row of zeros: the output is
    the others' alone."""
    n = 400
    q, kc, vc, table, q_start, kv_len = ref.paged_inputs([m, m], [n, 290], 8, 2, D, 16, dtype)
    q = torch.zeros_like(q)
    q[..., 0] = 8.0
    q[..., 1] = 1.0
    kc[..., 0] = 0.0
    kc[table[:, sink // 16].long(), sink % 16, :, 0] = nats * D**0.5 / 8.0
    vc += 100.0
    vc[table[:, sink // 16].long(), sink % 16] = 0.0
    (k8, ks), (v8, vs) = qc.quantised(kc), qc.quantised(vc)
    run((q, k8, v8, ks, vs, table, q_start, kv_len))


@pytest.mark.parametrize("e", [-30, 30, 60])
@pytest.mark.parametrize("m", [1, 70])
def test_value_scales_of_any_size(m, e):
    """Values of 2^e, and pages of other sizes beside ordinary ones."""
    q, k8, v8, ks, vs, *rest = qc.paged_inputs([m, m], [150, 300], 4, 2, 128, 16, BF)
    x = (q, k8, v8, ks, vs * 2.0**e, *rest)
    out = op(*x)
    want, size = qc.attend(x, ref.default_scale(128))
    ref.attention_close((out.double() * 2.0**-e), want * 2.0**-e, size * 2.0**-e, BF)
    vs = vs.clone()
    vs[rest[0][1, 5].long()] *= 2.0**20   # a page far above the others
    vs[rest[0][1, 9].long()] *= 2.0**-20
    run((q, k8, v8, ks, vs, *rest))


@pytest.mark.parametrize("scale", [2.0**-100, 2.0**-20, 2.0**20, 2.0**100])
@pytest.mark.parametrize("m", [1, 70])
def test_far_magnitudes_of_bf16_queries(m, scale):
    """Rows beyond f16's range either way, scaled back by `scale`; a row of zeros."""
    q, *rest = qc.paged_inputs([m, 1], [200, 60], 8, 2, 64, 16, BF)
    q = (q.double() * scale).to(BF)
    q[0, 0] = 0
    run((q, *rest), scale=0.125 / scale)


@pytest.mark.parametrize("dtype", [HF, BF])
@pytest.mark.parametrize("m", [1, 70])
def test_key_scales_of_any_size(m, dtype):
    """Keys of 1e30 and of 1e-30."""
    q, k8, v8, ks, vs, *rest = qc.paged_inputs([m], [150], 4, 2, 128, 16, dtype)
    run((q, k8, v8, ks * 2.0**100, vs, *rest), scale=2.0**-100 * 0.1)
    run((q, k8, v8, ks * 2.0**-100, vs, *rest), scale=2.0**100 * 0.1)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("q,n,H,hkv", [(65, 65, 8, 2), (130, 400, 4, 4), (257, 257, 8, 1), (100, 1000, 14, 2),
                                       (300, 301, 3, 1)])
def test_prompts(q, n, H, hkv, D):
    run(qc.paged_inputs([q, 1, q // 3], [n, n // 2, q], H, hkv, D, 16, BF))


@pytest.mark.parametrize("softcap,window", [(30.0, 0), (0.0, 50), (20.0, 200), (500.0, 0)])
def test_prompts_with_caps_and_windows(softcap, window):
    run(qc.paged_inputs([200, 1, 90], [333, 250, 90], 8, 2, 128, 16, BF, window=window), softcap, window)


def test_one_long_sequence_is_spread_and_joined():
    run(qc.paged_inputs([1], [9001], 8, 2, 128, 16, BF))
    run(qc.paged_inputs([2, 1], [5000, 3], 8, 8, 64, 32, HF))


def test_many_sequences():
    ns = [1 + (i * 37) % 50 for i in range(1300)]
    run(qc.paged_inputs([1] * len(ns), ns, 2, 1, 64, 16, BF))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("seqs,H,hkv,max_q", [(20, 32, 4, 0), (48, 16, 2, 1), (200, 16, 2, 0)])
def test_long_sequences_among_short_ones(seqs, H, hkv, max_q, D):
    ns = [i % 7 for i in range(seqs)]
    ns[3], ns[seqs // 2] = 6000, 700
    qs = [1] * seqs
    qs[3] = qs[4] = 3
    ns[4] = 2  # one of the three without keys
    run(qc.paged_inputs(qs, ns, H, hkv, D, 16, BF), max_q=max_q)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("steps", [1, 3, 4, 5, 8, 12])
def test_units_of_whole_warps_and_ctas(steps, D):
    """As many equal units as CTAs, of 32-key steps."""
    ctas = 2 * torch.cuda.get_device_properties(0).multi_processor_count
    run(qc.paged_inputs([1] * (ctas // 4), [32 * steps * 4] * (ctas // 4), 4, 1, D, 16, BF))


@pytest.mark.parametrize("H,hkv,D", [(8, 1, 128), (16, 1, 64), (5, 1, 128)])
def test_one_sequence_of_one_key_head(H, hkv, D):
    run(qc.paged_inputs([1], [30000], H, hkv, D, 16, BF))


@pytest.mark.parametrize("D,seqs", [(128, 8), (64, 16), (128, 260)])
@pytest.mark.parametrize("keys", [60, 4000])
def test_two_row_blocks_a_sequence(D, seqs, keys):
    """Sequences of 17 to 32 rows among shorter and longer ones, in either kernel."""
    qs = [(5, 8, 1, 6)[b % 4] for b in range(seqs)]
    ns = [keys if seqs < 100 else 90] * seqs
    qs[1], ns[2], ns[5] = 11, 0, 3
    *head, table, q_start, kv_len = qc.paged_inputs(qs, ns, 32, 8, D, 16, BF, pad=3)
    wide = torch.full((seqs, 2000), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    for max_q in (0, 11):
        run((*head, wide, q_start, kv_len), max_q=max_q)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("q,n,H,hkv", [(64, 64, 8, 2), (1000, 1000, 4, 1), (33, 3000, 8, 8), (513, 700, 2, 2),
                                       (128, 128, 2, 1), (2000, 100, 2, 1)])
def test_tile_units(q, n, H, hkv, D, dtype):
    run(qc.paged_inputs([q], [n], H, hkv, D, 16, dtype))


def test_prompts_and_single_tokens_in_one_batch():
    qs = [1, 500, 1, 3, 77, 0, 1, 260]
    ns = [900, 600, 1, 40, 77, 12, 2000, 260]
    run(qc.paged_inputs(qs, ns, 16, 2, 128, 16, BF, pad=9))
    run(qc.paged_inputs(qs, ns, 16, 2, 128, 16, BF, pad=9), max_q=500)
    run(qc.paged_inputs(qs, ns, 16, 2, 64, 16, HF), max_q=7)  # a hint that is too small


def test_many_prompts():
    qs = [9 + (i * 13) % 40 for i in range(300)]
    run(qc.paged_inputs(qs, [n + (i % 7) * 30 for i, n in enumerate(qs)], 8, 1, 64, 16, BF))


@pytest.mark.parametrize("m", [1, 90])
def test_strided_queries(m):
    q, *rest = qc.paged_inputs([m, 5, 2], [100, 60, 2], 8, 2, 64, 16, BF)
    wide = torch.zeros(q.shape[0], 12, 64, device="cuda", dtype=BF)
    wide[:, 3:11] = q
    run((wide[:, 3:11], *rest))
    run((q.transpose(0, 1).contiguous().transpose(0, 1), *rest))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("m", [1, 200])
@pytest.mark.parametrize("key", [0, 6, 31, 64, 150, 199])
@pytest.mark.parametrize("what", ["k", "k_scale", "v", "v_scale"])
def test_a_nan_reaches_every_row_that_sees_it(what, key, m, cap, D):
    q, k8, v8, ks, vs, table, q_start, kv_len = qc.paged_inputs([m], [200], 8, 2, D, 16, BF)
    clean = op(q, k8, v8, ks, vs, table, q_start, kv_len, 0.0, cap)
    at = table[0, key // 16].long(), key % 16
    if what in ("k", "v"):
        (k8 if what == "k" else v8).view(torch.uint8)[at][:, 3] = 0x7F
    else:
        (ks if what == "k_scale" else vs)[at] = float("nan")
    out = op(q, k8, v8, ks, vs, table, q_start, kv_len, 0.0, cap)
    seen = torch.arange(200 - m, 200, device="cuda") >= key
    if what == "v":
        assert out[seen][..., 3].isnan().all() and torch.equal(out[seen][..., 4:], clean[seen][..., 4:])
    else:
        assert out[seen].isnan().all()
    if what in ("k", "k_scale"):  # values that are hidden from a row must be finite for it
        assert torch.equal(out[~seen], clean[~seen])


def test_scales_of_zero():
    """Unwritten places of caches that began as zeros: keys and values of zero."""
    q, k8, v8, ks, vs, table, q_start, kv_len = qc.paged_inputs([1, 70], [40, 100], 8, 2, 64, 16, BF)
    pg = table[:, 1].long()
    k8.view(torch.uint8)[pg], v8.view(torch.uint8)[pg], ks[pg], vs[pg] = 0, 0, 0.0, 0.0
    run((q, k8, v8, ks, vs, table, q_start, kv_len))


def test_cache_offsets_past_32_bits():
    D, hkv, page = 128, 8, 128
    pages = 2**31 // (page * hkv * D) + 4
    k8, v8 = (torch.zeros(pages, page, hkv, D, device="cuda", dtype=torch.uint8).view(quant.E4M3) for _ in range(2))
    ks, vs = (torch.zeros(pages, page, hkv, device="cuda") for _ in range(2))
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32, device="cuda")
    for pg in table[0].tolist():
        for codes, scale in ((k8, ks), (v8, vs)):
            c, s = qc.quantised(torch.randn(page, hkv, D, device="cuda")[None])
            codes.view(torch.uint8)[pg], scale[pg] = c.view(torch.uint8)[0], s[0]
    small = [t[torch.tensor(table[0].tolist(), device="cuda")] if t.dtype != quant.E4M3
             else t.view(torch.uint8)[table[0].long()].view(quant.E4M3) for t in (k8, v8, ks, vs)]
    n = torch.tensor([2 * page + 50], dtype=torch.int32, device="cuda")
    for m in (1, 150):
        q = torch.randn(m, 8, D, device="cuda").to(BF)
        start = torch.tensor([0, m], dtype=torch.int32, device="cuda")
        out = op(q, k8, v8, ks, vs, table, start, n)
        near = torch.tensor([[0, 1, 2]], dtype=torch.int32, device="cuda")
        qc.attention_close(out, (q, *small, near, start, n), ref.default_scale(D))


@pytest.mark.parametrize("m", [1, 40])
def test_cache_offsets_past_64_gib(m):
    """Rows further apart than 2^32 times 16 bytes (the row kernel's other way to
    them), of a tensor of 75 GB of which three pages are touched; appended, then read."""
    if torch.cuda.mem_get_info()[0] < 90 << 30:
        pytest.skip("needs 90 GiB")
    D, hkv, page, far = 64, 2, 16, 37_500_000_000 // 4096 * 4096
    big = torch.empty(2 * far + (1 << 16), device="cuda", dtype=torch.uint8)
    sizes, strides = (3, page, hkv, D), (far, hkv * D, D, 1)
    k8, v8 = (big.as_strided(sizes, strides, o).view(quant.E4M3) for o in (0, 1 << 15))
    ks, vs = (torch.empty(3, page, hkv, device="cuda") for _ in range(2))
    n = 40
    g = torch.Generator("cuda").manual_seed(3)
    q, k, v = (torch.randn(n, h, D, device="cuda", generator=g).to(BF) for h in (8, hkv, hkv))
    one, none = torch.ones(1, 0, device="cuda"), torch.zeros(n, device="cuda", dtype=torch.int32)
    slots = torch.arange(n, device="cuda") + page * torch.tensor([2, 0, -2], device="cuda").repeat_interleave(page)[:n]
    torch.ops.b200.rope_append_quant(q, k, v, one, one, none, slots, k8, v8, ks, vs)
    i32 = dict(device="cuda", dtype=torch.int32)
    table, start, lens = torch.tensor([[2, 1, 0]], **i32), torch.tensor([0, m], **i32), torch.tensor([n], **i32)
    out = op(q[:m], k8, v8, ks, vs, table, start, lens)
    near = [torch.stack([c.view(torch.uint8)[i].clone() for i in range(3)]).view(quant.E4M3) for c in (k8, v8)]
    qc.attention_close(out, (q[:m], *near, ks, vs, table, start, lens), ref.default_scale(D))
    assert ((near[1].double() * vs.double()[..., None])[2, :page] - v[:page].double()).abs().max() < 0.2
    assert runtime.gemm_status() == 0
    del big, k8, v8
    torch.cuda.empty_cache()


def test_bad_indexes_are_reported_and_stay_in_bounds():
    *head, table, q_start, kv_len = qc.paged_inputs([1, 2], [40, 20], 8, 2, 64, 16, BF)
    for change in (lambda t, s, n: t.__setitem__((0, 1), 10**6), lambda t, s, n: t.__setitem__((1, 0), -5),
                   lambda t, s, n: n.__setitem__(0, 10**6), lambda t, s, n: n.__setitem__(1, -3),
                   lambda t, s, n: s.__setitem__(2, 50), lambda t, s, n: s.__setitem__(1, -2)):
        t, s, n = table.clamp_min(0), q_start.clone(), kv_len.clone()
        change(t, s, n)
        runtime.gemm_status()
        op(*head, t, s, n)
        assert runtime.gemm_status() == 9
    run((*head, table, q_start, kv_len))


def test_empty_calls():
    q, *caches, table, q_start, kv_len = qc.paged_inputs([1, 2], [40, 20], 8, 2, 64, 16, BF)
    assert op(q[:0], *caches, table, q_start * 0, kv_len).shape == (0, 8, 64)
    out = op(q, *caches, table[:0], q_start[:1], kv_len[:0])
    assert out.shape == q.shape and out.abs().sum() == 0
    assert op(q, *caches, table[:, :0], q_start, kv_len * 0).abs().sum() == 0


def test_refusals():
    q, k8, v8, ks, vs, *rest = qc.paged_inputs([1, 2], [40, 20], 8, 2, 64, 16, BF)
    for bad in (lambda: op(q[:, :, :32], k8[..., :32], v8[..., :32], ks, vs, *rest),
                lambda: op(q[:, :7], k8, v8, ks, vs, *rest),
                lambda: op(q, k8.view(torch.uint8), v8.view(torch.uint8), ks, vs, *rest),
                lambda: op(q, k8.float().to(BF), v8.float().to(BF), ks, vs, *rest),
                lambda: op(q, k8, v8, ks[:1], vs[:1], *rest),
                lambda: op(q, k8, v8, ks, vs.contiguous(), *rest),
                lambda: op(q, k8, v8, ks.half(), vs.half(), *rest),
                lambda: op(q, k8, v8, ks.cpu(), vs.cpu(), *rest),
                lambda: op(q, k8, v8, ks, vs, *rest, 0.0, -1.0),
                lambda: op(q, k8, v8, ks, vs, *rest, 0.0, 0.0, -1),
                lambda: op(q.float(), k8, v8, ks, vs, *rest),
                lambda: op(q.clone().requires_grad_(), k8, v8, ks, vs, *rest)):
        with pytest.raises(RuntimeError):
            bad()


def test_two_graphs_and_two_streams():
    a = qc.paged_inputs([1] * 4, [700, 90, 2000, 5], 8, 2, 128, 16, BF, seed=1)
    b = qc.paged_inputs([3, 3, 300, 3], [70, 900, 300, 1500], 8, 2, 128, 16, BF, seed=2)
    want_a, want_b = op(*a), op(*b)
    graphs, outs = [], []
    for x in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(op(*x))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        op(*b)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want_a) and torch.equal(outs[1], want_b)


def test_a_replayed_graph_follows_its_index_tensors():
    x = qc.paged_inputs([1, 1], [200, 300], 8, 2, 64, 16, BF)
    op(*x)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = op(*x)
    for lens in ([1, 300], [200, 16], [0, 77]):
        x[7].copy_(torch.tensor(lens, dtype=torch.int32))
        g.replay()
        qc.attention_close(out, x, ref.default_scale(64))


def test_results_repeat_bit_for_bit():
    x = qc.paged_inputs([1, 5, 1, 40], [3000, 900, 1, 600], 8, 2, 128, 16, BF)
    first = op(*x)
    for _ in range(5):
        assert torch.equal(op(*x), first)


def test_c_abi():
    x = qc.paged_inputs([1, 20], [500, 20], 8, 2, 128, 16, HF)
    out = torch.full_like(x[0], float("nan"))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    cabi.paged_attention_quant(*x, out, status=status)
    assert status.item() == 0
    qc.attention_close(out, x, ref.default_scale(128))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
def test_stalled_wait_times_out_and_context_survives(D, dtype):
    x = qc.paged_inputs([300], [300], 4, 4, D, 16, dtype)
    out = torch.zeros_like(x[0])
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    cabi.paged_attention_quant(*x, out, status=status, timeout_ns=50_000_000, test_flags=cabi.PAGED_TEST_WITHHOLD_SCORES)
    torch.cuda.synchronize()
    assert status.item() == 6
    status.zero_()
    cabi.paged_attention_quant(*x, out, status=status)
    assert status.item() == 0
    qc.attention_close(out, x, ref.default_scale(D))


@pytest.mark.parametrize("D", [64, 128])
def test_a_q_start_that_runs_backwards_stays_inside_the_workspace(D):
    q, *caches, table, _, _ = qc.paged_inputs([300], [300], 4, 2, D, 16, BF)
    seqs = 64
    table = table.clamp_min(0).expand(seqs, -1).contiguous()
    q_start = torch.tensor([0, 300] * (seqs // 2) + [0], dtype=torch.int32, device="cuda")
    kv_len = torch.full((seqs,), 300, dtype=torch.int32, device="cuda")
    out, status = torch.empty_like(q), torch.zeros(1, dtype=torch.int32, device="cuda")
    need = cabi.paged_attention_quant(q, *caches, table, q_start, kv_len, out, status=status)
    ws = torch.full((need + (1 << 20),), 0x5a, dtype=torch.uint8, device="cuda")
    status.zero_()
    cabi.paged_attention_quant(q, *caches, table, q_start, kv_len, out, status=status, workspace=ws)
    assert status.item() == 9
    assert (ws[need:] == 0x5a).all()
