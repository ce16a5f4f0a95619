"""b200::paged_attention against the formula in 64 bits (the bound is
derived at serving_reference.attention_close).  Everything of the caches that
no query may see holds NaN, and tables name no page that is not needed, so a
read outside the mask shows in the output or in the status word."""
import os
import subprocess
import sys

import pytest
import torch

import serving_reference as ref
from compiler import runtime
from compiler.runtime import cabi

pytestmark = pytest.mark.gpu
runtime.load()
BF, HF = torch.bfloat16, torch.float16


def run(inputs, softcap=0.0, window=0, max_q=0, scale=0.0):
    q = inputs[0]
    runtime.gemm_status()
    out = torch.ops.b200.paged_attention(*inputs, scale, softcap, window, max_q)
    want, size = ref.paged_attention(*inputs, scale or ref.default_scale(q.shape[2]), softcap, window)
    ref.attention_close(out, want, size, q.dtype)
    end = int(inputs[4][-1])
    assert out[end:].abs().sum() == 0
    assert runtime.gemm_status() == 0
    return out


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,hkv", [(32, 8), (8, 8), (8, 1), (7, 1), (28, 4), (40, 1), (6, 2)])
def test_single_tokens(H, hkv, D, dtype):
    ns = [1, 2, 15, 16, 17, 100, 333, 1, 64]
    run(ref.paged_inputs([1] * len(ns), ns, H, hkv, D, 16, dtype))


@pytest.mark.parametrize("page", [1, 3, 16, 24, 64, 100, 128])
def test_page_sizes(page):
    ns = [1, page, page + 1, 200, 3 * page - 1, 77]
    ns = [max(1, n) for n in ns]
    run(ref.paged_inputs([1] * len(ns), ns, 8, 2, 64, page, BF))


@pytest.mark.parametrize("layout", ["nhd", "hnd", "pair"])
@pytest.mark.parametrize("D", [64, 128])
def test_cache_layouts(layout, D):
    run(ref.paged_inputs([1, 4, 1], [100, 50, 7], 8, 2, D, 16, BF, layout=layout))


@pytest.mark.parametrize("softcap,window", [(30.0, 0), (5.0, 0), (0.0, 1), (0.0, 17), (0.0, 100), (50.0, 33),
                                            (0.0, 10**6)])
@pytest.mark.parametrize("D", [64, 128])
def test_caps_and_windows(softcap, window, D):
    qs, ns = [1, 3, 1, 8, 20], [90, 200, 5, 8, 300]
    run(ref.paged_inputs(qs, ns, 8, 2, D, 16, BF, window=window), softcap, window)


@pytest.mark.parametrize("max_q", [0, 1, 33])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
def test_ragged_queries_and_rows_without_keys(D, dtype, max_q):
    # no queries, no keys, fewer keys than queries, and rows behind the last sequence
    qs = [0, 1, 3, 33, 5, 4, 0, 2]
    ns = [10, 40, 0, 33, 200, 2, 0, 2]
    out = run(ref.paged_inputs(qs, ns, 8, 2, D, 16, dtype, pad=5), max_q=max_q)
    assert out[1:4].abs().sum() == 0                       # kv_len 0
    start = sum(qs[:5])
    assert out[start:start + 2].abs().sum() == 0           # positions before the first key
    assert out[start + 2:start + 4].abs().sum() > 0


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("q,n,H,hkv", [(65, 65, 8, 2), (130, 400, 4, 4), (257, 257, 8, 1), (100, 1000, 14, 2),
                                       (300, 301, 3, 1)])
def test_prompts(q, n, H, hkv, D):
    run(ref.paged_inputs([q, 1, q // 3], [n, n // 2, q], H, hkv, D, 16, BF))


@pytest.mark.parametrize("softcap,window", [(30.0, 0), (0.0, 50), (20.0, 200)])
def test_prompts_with_caps_and_windows(softcap, window):
    run(ref.paged_inputs([200, 1, 90], [333, 250, 90], 8, 2, 128, 16, BF, window=window), softcap, window)


def test_one_long_sequence_is_spread_and_joined():
    run(ref.paged_inputs([1], [9001], 8, 2, 128, 16, BF))
    run(ref.paged_inputs([2, 1], [5000, 3], 8, 8, 64, 32, HF))


def test_many_sequences():
    """More sequences than a warp's lanes and than workers, short and ragged."""
    ns = [1 + (i * 37) % 50 for i in range(1300)]
    run(ref.paged_inputs([1] * len(ns), ns, 2, 1, 64, 16, BF))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("seqs,H,hkv,max_q", [(20, 32, 4, 0), (48, 16, 2, 1), (200, 16, 2, 0)])
def test_long_sequences_among_short_ones(seqs, H, hkv, max_q, D):
    """Rows of one part and of hundreds in one call, as the join's warps share
    them out: a CTA's own rows and those of all its warps, up to 32 sequences
    and more, more rows than one a warp side by side (max_q 1, 3 queries)."""
    ns = [i % 7 for i in range(seqs)]
    ns[3], ns[seqs // 2] = 6000, 700
    qs = [1] * seqs
    qs[3] = qs[4] = 3
    ns[4] = 2  # one of the three without keys
    run(ref.paged_inputs(qs, ns, H, hkv, D, 16, BF), max_q=max_q)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("steps", [1, 3, 4, 5, 8, 12])
def test_units_of_whole_warps_and_ctas(steps, D):
    """As many equal units as CTAs, of 16-key steps: a warp's run, parts of a
    CTA's, exactly a CTA's, and more."""
    ctas = 2 * torch.cuda.get_device_properties(0).multi_processor_count
    run(ref.paged_inputs([1] * ctas, [16 * steps] * ctas, 4, 1, D, 16, BF))
    run(ref.paged_inputs([1] * (ctas // 8), [16 * steps * 8] * (ctas // 8), 4, 1, D, 16, BF))


@pytest.mark.parametrize("H,hkv,D", [(8, 1, 128), (16, 1, 64), (32, 1, 128), (5, 1, 128)])
def test_one_sequence_of_one_key_head(H, hkv, D):
    """A unit of thousands of steps: a part a CTA, a bounded number of CTAs."""
    run(ref.paged_inputs([1], [30000], H, hkv, D, 16, BF))
    run(ref.paged_inputs([1, 1], [20011, 64], H, hkv, D, 16, BF))


@pytest.mark.parametrize("D,seqs", [(128, 8), (64, 16), (128, 260)])
@pytest.mark.parametrize("keys", [60, 4000])
def test_two_row_blocks_a_sequence(D, seqs, keys):
    """Sequences of 17 to 32 rows among shorter and longer ones: the row kernel
    for few keys (a wide table, so that many are possible) and for many
    sequences, the tile kernel for many keys."""
    qs = [(5, 8, 1, 6)[b % 4] for b in range(seqs)]
    ns = [keys if seqs < 100 else 90] * seqs
    qs[1], ns[2], ns[5] = 11, 0, 3
    q, kc, vc, table, q_start, kv_len = ref.paged_inputs(qs, ns, 32, 8, D, 16, BF, pad=3)
    wide = torch.full((seqs, 2000), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    for max_q in (0, 11):
        run((q, kc, vc, wide, q_start, kv_len), max_q=max_q)
    q8 = [min(m, 8) for m in qs]
    first = run(ref.paged_inputs(q8, ns, 32, 8, D, 16, BF), max_q=8)
    assert torch.equal(run(ref.paged_inputs(q8, ns, 32, 8, D, 16, BF), max_q=8), first)


def test_strided_queries():
    q, *rest = ref.paged_inputs([1, 5, 2], [30, 60, 2], 8, 2, 64, 16, BF)
    wide = torch.zeros(q.shape[0], 12, 64, device="cuda", dtype=BF)
    wide[:, 3:11] = q
    run((wide[:, 3:11], *rest))
    turned = q.transpose(0, 1).contiguous().transpose(0, 1)
    run((turned, *rest))


def test_large_scores_stay_finite():
    q, kc, vc, *rest = ref.paged_inputs([1, 3], [50, 20], 4, 2, 64, 16, BF)
    out = torch.ops.b200.paged_attention(q * 1000, kc, vc, *rest)
    assert out.isfinite().all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("m", [1, 200])
@pytest.mark.parametrize("key", [0, 6, 7, 64, 71, 150, 199])
def test_a_nan_key_reaches_every_row_that_sees_it_and_no_other(key, m, cap, D):
    q, kc, vc, table, q_start, kv_len = ref.paged_inputs([m], [200], 8, 2, D, 16, BF)
    op = torch.ops.b200.paged_attention
    clean = op(q, kc, vc, table, q_start, kv_len, 0.0, cap)
    kc = kc.clone()
    kc[table[0, key // 16], key % 16, :, 3] = float("nan")
    out = op(q, kc, vc, table, q_start, kv_len, 0.0, cap)
    seen = torch.arange(200 - m, 200, device="cuda") >= key
    assert out[seen].isnan().all() and torch.equal(out[~seen], clean[~seen])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("m", [1, 200])
@pytest.mark.parametrize("key", [0, 6, 64, 71, 199])
def test_an_infinite_score(key, m, D):
    """+inf - inf is NaN in the softmax; a score of -inf has no weight."""
    q, kc, vc, table, q_start, kv_len = ref.paged_inputs([m], [200], 8, 2, D, 16, BF)
    seen = (torch.arange(200 - m, 200, device="cuda") >= key)[:, None]
    at = table[0, key // 16], key % 16
    lone = torch.arange(200 - m, 200, device="cuda")[:, None] == 0  # sees this key alone when key == 0
    kc = kc.clone()
    kc[at][:, 3] = float("inf")
    out = torch.ops.b200.paged_attention(q, kc, vc, table, q_start, kv_len)
    up, down = seen & (q[..., 3] > 0), seen & (q[..., 3] < 0)
    assert out[up].isnan().all()
    assert out[down & ~(lone & (key == 0))].isfinite().all() and out[~seen.expand(-1, 8)].isfinite().all()
    kc[at][:, 3] = float(2**15)  # -2^15 |q|: no weight either
    want = torch.ops.b200.paged_attention(q, kc, vc, table, q_start, kv_len)
    keep = down & (q[..., 3] < -0.1) & ~(lone & (key == 0))
    torch.testing.assert_close(out[keep], want[keep], rtol=2.0**-7, atol=2.0**-7)


def test_cache_offsets_past_32_bits():
    D, hkv, page = 128, 8, 128
    pages = 2**31 // (page * hkv * D) + 4
    kc, vc = (torch.zeros(pages, page, hkv, D, device="cuda", dtype=BF) for _ in range(2))
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32, device="cuda")
    for pg in table[0].tolist():
        kc[pg].normal_()
        vc[pg].normal_()
    n = 2 * page + 50
    for m in (1, 150):
        q = torch.randn(m, 8, D, device="cuda").to(BF)
        run((q, kc, vc, table, torch.tensor([0, m], dtype=torch.int32, device="cuda"),
             torch.tensor([n], dtype=torch.int32, device="cuda")))


def test_bad_indexes_are_reported_and_stay_in_bounds():
    q, kc, vc, table, q_start, kv_len = ref.paged_inputs([1, 2], [40, 20], 8, 2, 64, 16, BF)
    for change in (lambda t, s, n: t.__setitem__((0, 1), 10**6), lambda t, s, n: t.__setitem__((1, 0), -5),
                   lambda t, s, n: n.__setitem__(0, 10**6), lambda t, s, n: n.__setitem__(1, -3),
                   lambda t, s, n: s.__setitem__(2, 50), lambda t, s, n: s.__setitem__(1, -2)):
        t, s, n = table.clamp_min(0), q_start.clone(), kv_len.clone()
        change(t, s, n)
        runtime.gemm_status()
        torch.ops.b200.paged_attention(q, kc, vc, t, s, n)
        assert runtime.gemm_status() == 9
    run((q, kc, vc, table, q_start, kv_len))


def test_empty_calls():
    q, kc, vc, table, q_start, kv_len = ref.paged_inputs([1, 2], [40, 20], 8, 2, 64, 16, BF)
    op = torch.ops.b200.paged_attention
    assert op(q[:0], kc, vc, table, q_start * 0, kv_len).shape == (0, 8, 64)
    out = op(q, kc, vc, table[:0], q_start[:1], kv_len[:0])
    assert out.shape == q.shape and out.abs().sum() == 0
    assert op(q, kc, vc, table[:, :0], q_start, kv_len * 0).abs().sum() == 0


def test_refusals():
    q, kc, vc, table, q_start, kv_len = ref.paged_inputs([1, 2], [40, 20], 8, 2, 64, 16, BF)
    op = torch.ops.b200.paged_attention
    for bad in (lambda: op(q[:, :, :32], kc[..., :32], vc[..., :32], table, q_start, kv_len),
                lambda: op(q[:, :7], kc, vc, table, q_start, kv_len),
                lambda: op(q.half(), kc, vc, table, q_start, kv_len),
                lambda: op(q, kc, vc[:1], table, q_start, kv_len),
                lambda: op(q, kc, vc, table.long(), q_start, kv_len),
                lambda: op(q, kc, vc, table, q_start[:2], kv_len),
                lambda: op(q, kc, vc, table[:1], q_start, kv_len),
                lambda: op(q, kc, vc, table, q_start, kv_len.cpu()),
                lambda: op(q, kc, vc, table, q_start, kv_len, 0.0, -1.0),
                lambda: op(q, kc, vc, table, q_start, kv_len, 0.0, 0.0, -1),
                lambda: op(q.float(), kc.float(), vc.float(), table, q_start, kv_len),
                lambda: op(q.clone().requires_grad_(), kc, vc, table, q_start, kv_len)):
        with pytest.raises(RuntimeError):
            bad()


def test_two_graphs_and_two_streams():
    """Two captured graphs replayed on two streams at once, and eager calls
    between them, keep to their own workspaces."""
    a = ref.paged_inputs([1] * 4, [700, 90, 2000, 5], 8, 2, 128, 16, BF, seed=1)
    b = ref.paged_inputs([3] * 4, [70, 900, 20, 1500], 8, 2, 128, 16, BF, seed=2)
    op = torch.ops.b200.paged_attention
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
    q, kc, vc, table, q_start, kv_len = ref.paged_inputs([1, 1], [200, 300], 8, 2, 64, 16, BF)
    op = torch.ops.b200.paged_attention
    op(q, kc, vc, table, q_start, kv_len)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = op(q, kc, vc, table, q_start, kv_len)
    for lens in ([1, 300], [200, 16], [0, 77]):
        kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        g.replay()
        want, size = ref.paged_attention(q, kc, vc, table, q_start, kv_len, ref.default_scale(64))
        ref.attention_close(out, want, size, BF)


def test_results_repeat_bit_for_bit():
    x = ref.paged_inputs([1, 5, 1, 40], [3000, 900, 1, 600], 8, 2, 128, 16, BF)
    first = torch.ops.b200.paged_attention(*x)
    for _ in range(5):
        assert torch.equal(torch.ops.b200.paged_attention(*x), first)


def test_c_abi():
    x = ref.paged_inputs([1, 20], [500, 20], 8, 2, 128, 16, HF)
    out = torch.full_like(x[0], float("nan"))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    cabi.paged_attention(*x, out, status=status)
    assert status.item() == 0
    want, size = ref.paged_attention(*x, ref.default_scale(128))
    ref.attention_close(out, want, size, HF)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("q,n,H,hkv", [(64, 64, 8, 2), (1000, 1000, 4, 1), (33, 3000, 8, 8), (513, 700, 2, 2),
                                       (128, 128, 2, 1), (2000, 100, 2, 1)])
def test_tile_units(q, n, H, hkv, D, dtype):
    """Whole and cut units, blocks that end inside a tile, causal tiles of
    different lengths, more queries than keys."""
    run(ref.paged_inputs([q], [n], H, hkv, D, 16, dtype))


def test_prompts_and_single_tokens_in_one_batch():
    qs = [1, 500, 1, 3, 77, 0, 1, 260]
    ns = [900, 600, 1, 40, 77, 12, 2000, 260]
    run(ref.paged_inputs(qs, ns, 16, 2, 128, 16, BF, pad=9))
    run(ref.paged_inputs(qs, ns, 16, 2, 128, 16, BF, pad=9), max_q=500)
    run(ref.paged_inputs(qs, ns, 16, 2, 64, 16, HF), max_q=7)  # a hint that is too small


def test_many_prompts():
    qs = [9 + (i * 13) % 40 for i in range(300)]
    run(ref.paged_inputs(qs, [n + (i % 7) * 30 for i, n in enumerate(qs)], 8, 1, 64, 16, BF))


def test_stalled_wait_times_out_and_context_survives():
    """The test hook withholds the first score block's signal: a wait runs out
    after 50 ms, the kernel reports B200K_ERR_TIMEOUT, drains and returns,
    and the next call is right."""
    x = ref.paged_inputs([300], [300], 4, 4, 128, 16, BF)
    out = torch.zeros_like(x[0])
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    cabi.paged_attention(*x, out, status=status, timeout_ns=50_000_000, test_flags=cabi.PAGED_TEST_WITHHOLD_SCORES)
    torch.cuda.synchronize()
    assert status.item() == 6
    status.zero_()
    cabi.paged_attention(*x, out, status=status)
    assert status.item() == 0
    want, size = ref.paged_attention(*x, ref.default_scale(128))
    ref.attention_close(out, want, size, BF)


@pytest.mark.parametrize("D", [64, 128])
def test_a_q_start_that_runs_backwards_stays_inside_the_workspace(D):
    """Every other sequence claims all tokens: many times the 256-row blocks
    that the workspace is sized for.  Reported, and nothing past it written."""
    q, kc, vc, table, _, _ = ref.paged_inputs([300], [300], 4, 2, D, 16, BF)
    seqs = 64
    table = table.clamp_min(0).expand(seqs, -1).contiguous()
    q_start = torch.tensor([0, 300] * (seqs // 2) + [0], dtype=torch.int32, device="cuda")
    kv_len = torch.full((seqs,), 300, dtype=torch.int32, device="cuda")
    out, status = torch.empty_like(q), torch.zeros(1, dtype=torch.int32, device="cuda")
    need = cabi.paged_attention(q, kc, vc, table, q_start, kv_len, out, status=status)
    ws = torch.full((need + (1 << 20),), 0x5a, dtype=torch.uint8, device="cuda")
    status.zero_()
    cabi.paged_attention(q, kc, vc, table, q_start, kv_len, out, status=status, workspace=ws)
    assert status.item() == 9
    assert (ws[need:] == 0x5a).all()


def test_strides_of_dims_of_one_element_do_not_matter():
    q, kc, vc, table, q_start, kv_len = ref.paged_inputs([1], [40], 1, 1, 64, 16, BF)
    one = lambda t: t.as_strided(t.shape, tuple(s if n > 1 else 7 for n, s in zip(t.shape, t.stride())))  # noqa: E731
    want = torch.ops.b200.paged_attention(q, kc, vc, table, q_start, kv_len)
    got = torch.ops.b200.paged_attention(one(q), one(kc), vc, one(table), q_start, kv_len)
    assert torch.equal(got, want)


def test_a_first_call_inside_a_capture():
    """A process whose first paged_attention calls (both kernels) are being
    captured: no status word exists yet, no attribute is set."""
    code = """
import sys; sys.path[:0] = [%r, %r]
import torch, serving_reference as ref
from compiler import runtime
runtime.load()
x = ref.paged_inputs([1, 300], [90, 300], 8, 2, 64, 16, torch.bfloat16)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = torch.ops.b200.paged_attention(*x)
g.replay()
want, size = ref.paged_attention(*x, ref.default_scale(64))
ref.attention_close(out, want, size, torch.bfloat16)
print("fine")
""" % (os.path.dirname(ref.__file__), os.path.dirname(os.path.dirname(os.path.dirname(cabi.__file__))))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-2000:]
