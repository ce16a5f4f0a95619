"""Plain 64-bit forms of the paged-cache serving operators, and inputs for
their tests: paged caches whose unused places hold NaN."""
from __future__ import annotations

import math

import torch

HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


def add_rms_norm(x, residual, weight, eps, plus_one=False):
    """(sum in x's type, y in 64 bits)."""
    total = (x.double() + residual.double()).to(x.dtype)
    h = total.double()
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * (weight.double() + (1.0 if plus_one else 0.0))
    return total, y


def rotate(x, cos, sin):
    """Rotate-half embedding of x [t, heads, d], tables [t, R/2]; returns the
    result and the sum of the products' magnitudes, in 64 bits."""
    half = cos.shape[1]
    x = x.double()
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    c, s = cos.double()[:, None], sin.double()[:, None]
    y = torch.cat([a * c - b * s, b * c + a * s, rest], -1)
    size = torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs(), rest * 0], -1)
    return y, size


def paged_attention(q, k_cache, v_cache, table, q_start, kv_len, scale, softcap=0.0, window=0):
    """(out, sum_j p_j |v_j|) in 64 bits, one sequence at a time."""
    T, H, D = q.shape
    page, hkv = k_cache.shape[1], k_cache.shape[2]
    G = H // hkv
    out = torch.zeros(T, H, D, dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    starts, lens = q_start.tolist(), kv_len.tolist()
    for b, n in enumerate(lens):
        m = starts[b + 1] - starts[b]
        for i in range(m):
            pos = n - m + i
            lo = max(0, pos - window + 1) if window else 0
            if pos < lo or pos < 0:
                continue
            keys = torch.arange(lo, pos + 1, device=q.device)
            pages = table[b, keys // page].long()
            k = k_cache[pages, keys % page].double()  # [keys, hkv, d]
            v = v_cache[pages, keys % page].double()
            x = torch.einsum("hgd,nhd->hgn", q[starts[b] + i].double().unflatten(0, (hkv, G)), k) * scale
            if softcap:
                x = softcap * torch.tanh(x / softcap)
            p = torch.softmax(x, -1)
            out[starts[b] + i] = torch.einsum("hgn,nhd->hgd", p, v).flatten(0, 1)
            size[starts[b] + i] = torch.einsum("hgn,nhd->hgd", p, v.abs()).flatten(0, 1)
    return out, size


def attention_close(got, want, size, dtype):
    """Bound: each probability rounds to the input type (half a step of
    sum p |v|), the output rounds once (half a step of itself), and the fp32
    scores and sums add at most 5e-4 of sum p |v|: scores here stay below 64
    and sum at most 128 products, so an fp32 score is off by less than
    128 * 2^-24 * 32 = 2.4e-4, which moves a probability relative to the
    others by at most twice that."""
    h = HALF_STEP[dtype]
    bound = (h + 5e-4) * size + h * want.abs() + 1e-7
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert (err <= bound).all(), (err - bound).max().item()


def paged_inputs(qs, ns, H, hkv, D, page, dtype, seed=0, window=0, pad=0, layout="nhd", spare=3, device="cuda"):
    """Packed queries, caches and index tensors of sequences with `qs` queries
    and `ns` keys.  Every place of the caches that no query may see is NaN,
    and table entries of pages that are not needed are -1."""
    g = torch.Generator(device=device).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device=device, generator=g).to(dtype)

    used = [-(-n // page) for n in ns]
    pages = sum(used) + spare
    nan = float("nan")
    if layout == "nhd":
        kc, vc = (torch.full((pages, page, hkv, D), nan, device=device, dtype=dtype) for _ in range(2))
    elif layout == "hnd":
        kc, vc = (torch.full((pages, hkv, page, D), nan, device=device, dtype=dtype).transpose(1, 2) for _ in range(2))
    else:  # one tensor for both, keys and values of a page side by side
        both = torch.full((pages, 2, page, hkv, D), nan, device=device, dtype=dtype)
        kc, vc = both[:, 0], both[:, 1]
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(ns), max([1] + used) + 1), -1, dtype=torch.int32)
    at = 0
    for b, (m, n) in enumerate(zip(qs, ns)):
        lo = max(0, n - m - window + 1) if window else 0
        for i in range(used[b]):
            if m == 0 or (i + 1) * page <= lo:
                at += 1
                continue  # never read
            pg = order[at]
            at += 1
            table[b, i] = pg
            first, last = max(lo, i * page), min(n, (i + 1) * page)
            if last > first:
                kc[pg, first - i * page:last - i * page] = randn(last - first, hkv, D)
                vc[pg, first - i * page:last - i * page] = randn(last - first, hkv, D)
    starts = [0]
    for m in qs:
        starts.append(starts[-1] + m)
    q = randn(starts[-1] + pad, H, D) * 1.5
    return (q, kc, vc, table.to(device), torch.tensor(starts, dtype=torch.int32, device=device),
            torch.tensor(ns, dtype=torch.int32, device=device))


def default_scale(D):
    return 1.0 / math.sqrt(D)
